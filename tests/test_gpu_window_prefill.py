"""Attention of prompt chunks under a window with sinks, over fp16 and e4m3 caches, against
a 64-bit reference; cache rows that no query sees hold NaN."""
import math

import pytest
import torch

import _window_ref as ref

pytestmark = pytest.mark.gpu


def _ops():
    from vllm_apple_b200 import ops
    return ops


class Case:
    """Chunks on the host.  ``chunks``: (context before the chunk, new tokens) per sequence;
    ``pad`` rows of no sequence follow."""

    def __init__(self, Hq, Hkv, D, chunks, bs=16, layout="hnd", q8=False, window=0, sinks=0,
                 seed=0, pad=0):
        g = torch.Generator().manual_seed(seed)
        self.__dict__.update(Hq=Hq, Hkv=Hkv, D=D, chunks=chunks, bs=bs, layout=layout, q8=q8,
                             window=window, sinks=sinks, scale=1 / math.sqrt(D))
        self.lens = [a + b for a, b in chunks]
        self.start = [0]
        for _, n in chunks:
            self.start.append(self.start[-1] + n)
        need = [(n + bs - 1) // bs for n in self.lens]
        nb = max(sum(need), 1) + 2
        perm = torch.randperm(nb, generator=g).int()
        self.table = torch.full((len(chunks), max(max(need), 1)), 1 << 30, dtype=torch.int32)
        shape = (nb, Hkv, bs) if layout == "hnd" else (nb, bs, Hkv)
        kv = [torch.full(shape + (D,), 127 if q8 else math.nan,
                         dtype=torch.uint8 if q8 else torch.float16) for _ in range(2)]
        ex = [torch.randint(113, 135, shape, generator=g, dtype=torch.uint8) for _ in range(2)]
        at = 0
        for i, (ctx, new) in enumerate(chunks):
            n = self.lens[i]
            pos = torch.arange(n)
            first = max(ctx, 0)
            if new:
                lo = max(0, first - window + 1) if window > 0 else 0
                pos = pos[(pos >= lo) | (pos < sinks)]
            else:
                pos = pos[:0]
            pages = torch.zeros(need[i], dtype=torch.bool)
            pages[pos // bs] = True
            ids = perm[at:at + need[i]]
            self.table[i, :need[i]] = torch.where(pages, ids, -3)
            at += need[i]
            for c, e in zip(kv, ex):
                x = torch.randn(len(pos), Hkv, D, generator=g).half()
                b, o = ids.long()[pos // bs], pos % bs
                if q8:
                    codes, exps = ref.quantise(x)
                    ref.put_rows(c, b, o, codes, layout)
                    ref.put_rows(e, b, o, exps, layout)
                else:
                    ref.put_rows(c, b, o, x, layout)
        self.kv, self.ex = kv, ex if q8 else [None, None]
        self.q = torch.randn(self.start[-1] + pad, Hq, D, generator=g).half()

    def run(self, out=None, q=None, shift=0, **kw):
        kv = [c.cuda().view(torch.float8_e4m3fn) if self.q8 else c.cuda() for c in self.kv]
        ks, vs = (None if e is None else e.cuda() for e in self.ex)
        q = self.q.cuda() if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        _ops().paged_window_prefill(
            out, q, *kv, self.table.cuda(),
            torch.tensor(self.start, dtype=torch.int32).cuda() + shift,
            torch.tensor(self.lens, dtype=torch.int32).cuda(), scale=self.scale,
            window=self.window, sink_tokens=self.sinks, k_scale=ks, v_scale=vs,
            layout=self.layout, **kw)
        return out

    def cache_rows(self, i, pos):
        k, v = (ref.rows(c, self.table[i], pos, self.bs, self.layout) for c in self.kv)
        if self.q8:
            k, v = (ref.values(x, ref.rows(e, self.table[i], pos, self.bs, self.layout))
                    for x, e in zip((k, v), self.ex))
        return k, v

    def expected(self, i):
        ctx, new = self.chunks[i]
        pos = torch.arange(self.lens[i])
        lo = max(0, max(ctx, 0) - self.window + 1) if self.window > 0 else 0
        pos = pos[(pos >= lo) | (pos < self.sinks)]
        k, v = self.cache_rows(i, pos)
        skip = max(-ctx, 0)  # tokens before position 0
        q = self.q[self.start[i] + skip:self.start[i + 1]]
        return skip, ref.attend(q, k, v, ctx + skip, pos, self.window, self.sinks, self.scale)

    def check(self, out, only=None):
        out = out.cpu()
        for i, (ctx, new) in enumerate(self.chunks):
            if new == 0 or (only is not None and i not in only):
                continue
            rows = out[self.start[i]:self.start[i + 1]]
            if self.lens[i] <= 0:
                assert bool((rows == 7).all())
                continue
            skip, (o, t) = self.expected(i)
            assert bool((rows[:skip] == 7).all())
            err = (rows[skip:].double() - o).abs()
            assert bool((err <= t).all()), (
                f"sequence {i} {self.chunks[i]}: {float((err / t).max())} of the bound at "
                f"{(err > t).nonzero()[:4].tolist()}")
        assert bool((out[self.start[-1]:] == 7).all()), "a row of no sequence was written"


SHAPES = [(14, 2, 64), (32, 8, 128), (8, 8, 96), (12, 1, 32), (16, 1, 64), (3, 1, 128)]
CHUNKS = [(0, 1), (5, 130), (300, 1), (0, 0), (127, 3), (64, 64), (1, 257), (700, 40)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("window,sinks,bs,layout", [(0, 0, 16, "hnd"), (100, 4, 16, "nhd"),
                                                    (1, 0, 8, "hnd"), (129, 140, 5, "nhd")])
def test_prefill_matches_reference(Hq, Hkv, D, q8, window, sinks, bs, layout):
    c = Case(Hq, Hkv, D, CHUNKS, bs=bs, layout=layout, q8=q8, window=window, sinks=sinks,
             seed=Hq + D, pad=9)
    out = c.run()
    assert _ops().check_device_errors() == 0
    c.check(out)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("chunks,window,sinks,bs", [
    ([(0, 1)], 0, 0, 16), ([(0, 2)], 1, 1, 1), ([(0, 600)], 64, 4, 64), ([(2000, 300)], 1000, 3, 16),
    ([(3000, 20)], 512, 1500, 32), ([(1500, 129)], 1 << 30, 4, 128), ([(0, 1100)], 0, 0, 7),
    ([(1000, 1)] * 3, 128, 128, 16), ([(511, 257)], 256, 300, 256)])
def test_windows_and_sinks_across_tiles(chunks, window, sinks, bs, q8):
    c = Case(8, 2, 64, chunks, bs=bs, q8=q8, window=window, sinks=sinks, seed=len(chunks))
    out = c.run()
    assert torch.equal(out, c.run())
    assert _ops().check_device_errors() == 0
    c.check(out)


def test_group_of_128_heads_and_of_none_power_of_two():
    for Hq, Hkv in ((128, 1), (100, 1), (22, 2)):
        c = Case(Hq, Hkv, 64, [(200, 5), (0, 3)], window=150, sinks=2, seed=Hq)
        out = c.run()
        assert _ops().check_device_errors() == 0
        c.check(out)


@pytest.mark.parametrize("q8", [False, True])
def test_tokens_after_other_rows_and_views(q8):
    """query_start_loc that starts behind other rows (the decode rows of a batch), Q as a
    plane of a QKV buffer and out as a slice of a wider one."""
    c = Case(8, 2, 64, [(50, 70), (0, 33)], q8=q8, window=40, sinks=2, seed=4)
    T = c.q.shape[0]
    buf = torch.zeros(T + 3, 12, 64, dtype=torch.float16, device="cuda")
    buf[3:, 2:10] = c.q.cuda()
    out = torch.full((T + 3, 9, 72), 7.0, dtype=torch.float16, device="cuda")
    c.run(out=out[:, :8, :64], q=buf[:, 2:10], shift=3)
    assert _ops().check_device_errors() == 0
    c.check(out[3:, :8, :64])
    assert bool((out[:3] == 7).all() and (out[:, 8] == 7).all() and (out[..., 64:] == 7).all())


@pytest.mark.parametrize("q8", [False, True])
def test_masked_values_that_are_not_finite(q8):
    """K and V rows of a chunk that hold infinities or NaN reach exactly the tokens that
    see them: the tokens before them and those whose window has passed stay finite."""
    c = Case(4, 2, 64, [(10, 300)], q8=q8, window=60, sinks=0, seed=9)
    at = [(100, 5), (171, 60), (240, 0)]  # (position, column)
    for p, d in at:
        b, o = int(c.table[0, p // c.bs]), p % c.bs
        c.kv[1][b, :, o, d] = 127 if q8 else math.inf
    b, o = int(c.table[0, 200 // c.bs]), 200 % c.bs
    c.kv[0][b, :, o, 3] = 127 if q8 else math.nan
    out = c.run().cpu().double()
    assert _ops().check_device_errors() == 0
    clean = Case(4, 2, 64, [(10, 300)], q8=q8, window=60, sinks=0, seed=9)
    o, t = clean.expected(0)[1]
    p = 10 + torch.arange(300)
    seen_k = (p >= 200) & (p < 260)
    assert bool(torch.isnan(out[seen_k]).all())
    hit = torch.zeros(300, 64, dtype=torch.bool)
    for pos, d in at:
        hit[(p >= pos) & (p < pos + 60), d] = True
    want = hit & ~seen_k[:, None]
    got = out.transpose(1, 2)  # [token, D, head]
    assert bool((torch.isnan(got) if q8 else got == math.inf)[want].all())
    rest = ~hit & ~seen_k[:, None]
    err = (out - o).abs().transpose(1, 2)
    # the other columns of a row keep their values: the weights did not change
    assert bool((err <= t.transpose(1, 2))[rest].all())


def test_negative_positions_and_padding_are_left_alone():
    """A chunk with more tokens than its sequence has positions, and an empty sequence."""
    c = Case(8, 2, 64, [(-3, 10), (20, 5)], window=0, seed=2, pad=4)
    out = c.run()
    assert _ops().check_device_errors() == 0
    c.check(out)
    c = Case(8, 2, 64, [(0, 6), (20, 5)], window=0, seed=2)
    c.lens[0] = 0
    out = c.run()
    assert bool((out[:6] == 7).all())
    c.check(out, only=[1])


@pytest.mark.parametrize("q8", [False, True])
def test_bad_metadata_is_flagged_and_rows_left_alone(q8):
    ops = _ops()
    from vllm_apple_b200._lib import VA_FLAG_BAD_BLOCK, VA_FLAG_CTX_OVERFLOW
    c = Case(8, 2, 64, [(0, 300), (0, 40)], q8=q8, window=50, sinks=4, seed=3)
    good = c.table.clone()
    c.table[0, 8] = 10 ** 9  # positions 128..143: seen by tokens 128..192
    out = c.run()
    assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_BAD_BLOCK
    c.table = good
    assert bool((out[128:193] == 7).all())
    keep = torch.ones(340, dtype=torch.bool)
    keep[128:193] = False
    want = c.run()
    assert torch.equal(out[keep.cuda()], want[keep.cuda()])
    c.check(want)
    # a sequence longer than its table; tokens past the end of q
    c.table = good[:, :10].contiguous()
    out = c.run()
    assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_CTX_OVERFLOW
    assert bool((out[:300] == 7).all())
    c.check(out, only=[1])
    c.table = good
    out = c.run(shift=1)
    assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_CTX_OVERFLOW
    assert bool((out[301:] == 7).all())


@pytest.mark.parametrize("q8", [False, True])
def test_captured_calls_replay(q8):
    c = Case(32, 8, 128, [(100, 200), (0, 7)], q8=q8, window=64, sinks=4, seed=1)
    want = c.run()
    kv = [x.cuda().view(torch.float8_e4m3fn) if q8 else x.cuda() for x in c.kv]
    ks, vs = (None if e is None else e.cuda() for e in c.ex)
    q, table = c.q.cuda(), c.table.cuda()
    qsl = torch.tensor(c.start, dtype=torch.int32).cuda()
    sl = torch.tensor(c.lens, dtype=torch.int32).cuda()
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _ops().paged_window_prefill(out, q, *kv, table, qsl, sl, scale=c.scale, window=64,
                                    sink_tokens=4, k_scale=ks, v_scale=vs)
    out.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_one_token_chunks_agree_with_decode():
    """A chunk of one token is a decode step: both kernels are within their bounds of the
    same reference, on the same cache."""
    c = Case(32, 8, 128, [(99, 1), (0, 1), (1000, 1)], window=300, sinks=4, seed=7)
    c.check(c.run())
    out = torch.full_like(c.q, 7.0, device="cuda")
    _ops().paged_window_decode(out, c.q.cuda(), c.kv[0].cuda(), c.kv[1].cuda(), c.table.cuda(),
                               torch.tensor(c.lens, dtype=torch.int32).cuda(), scale=c.scale,
                               max_seq_len=1001, window=300, sink_tokens=4)
    c.check(out)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("bs,layout", [(16, "hnd"), (128, "nhd"), (24, "hnd")])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 1, 96)])
def test_cache_views(Hq, Hkv, D, bs, layout, q8):
    """K and V interleaved in one tensor whose blocks, heads and rows have gaps."""
    c = Case(Hq, Hkv, D, CHUNKS, bs=bs, layout=layout, q8=q8, window=200, sinks=5, seed=3)
    nb, d1, d2, _ = c.kv[0].shape
    big = torch.full((nb + 1, 2, d1 + 1, d2 + 1, D + 16), 127 if q8 else math.nan,
                     dtype=c.kv[0].dtype)
    for v in range(2):
        big[:nb, v, :d1, :d2, :D] = c.kv[v]
    big = big.cuda()
    views = [big[:nb, v, :d1, :d2, :D] for v in range(2)]
    if q8:
        views = [x.view(torch.float8_e4m3fn) for x in views]
    ks, vs = (None if e is None else e.cuda() for e in c.ex)
    q = c.q.cuda()
    out = torch.full_like(q, 7.0)
    _ops().paged_window_prefill(
        out, q, *views, c.table.cuda(), torch.tensor(c.start, dtype=torch.int32).cuda(),
        torch.tensor(c.lens, dtype=torch.int32).cuda(), scale=c.scale, window=200,
        sink_tokens=5, k_scale=ks, v_scale=vs, layout=layout)
    assert _ops().check_device_errors() == 0
    c.check(out)
