"""Single-token attention under a window with sinks, over fp16 and e4m3 caches, against a
64-bit reference; every cache row that no query sees holds NaN."""
import math

import pytest
import torch

import _window_ref as ref

pytestmark = pytest.mark.gpu


def _ops():
    from vllm_apple_b200 import ops
    return ops


class Case:
    """A decode batch on the host: caches whose unseen rows are NaN, and table entries of
    unread blocks that name no block."""

    def __init__(self, Hq, Hkv, D, lens, bs=16, layout="hnd", q8=False, window=0, sinks=0,
                 seed=0, new=True):
        g = torch.Generator().manual_seed(seed)
        self.__dict__.update(Hq=Hq, Hkv=Hkv, D=D, lens=lens, bs=bs, layout=layout, q8=q8,
                             window=window, sinks=sinks, scale=1 / math.sqrt(D))
        B = len(lens)
        need = [(n + bs - 1) // bs for n in lens]
        nb = max(sum(need) + 2, 1)
        perm = torch.randperm(nb, generator=g).int()
        self.table = torch.full((B, max(max(need), 1) + 1), 1 << 30, dtype=torch.int32)
        shape = (nb, Hkv, bs) if layout == "hnd" else (nb, bs, Hkv)
        kv = [torch.full(shape + (D,), 127 if q8 else math.nan,
                         dtype=torch.uint8 if q8 else torch.float16) for _ in range(2)]
        ex = [torch.randint(113, 135, shape, generator=g, dtype=torch.uint8) for _ in range(2)]
        at = 0
        for i, n in enumerate(lens):
            pos = torch.arange(n)
            see = ref.visible(n - 1, pos, window, sinks)
            pos = pos[see]
            pages = torch.zeros(need[i], dtype=torch.bool)
            pages[pos // bs] = True
            ids = perm[at:at + need[i]]
            self.table[i, :need[i]] = torch.where(pages, ids, -5)
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
        self.q = torch.randn(B, Hq, D, generator=g).half()
        self.new = [torch.randn(B, Hkv, D, generator=g).half() for _ in range(2)] if new else None
        if q8 and new:
            self.new[0][:, :, 0] *= 30

    def device_caches(self):
        kv = [c.cuda().view(torch.float8_e4m3fn) if self.q8 else c.cuda() for c in self.kv]
        return kv + [None if e is None else e.cuda() for e in self.ex]

    def write_new(self):
        """The new rows into the host caches."""
        for i, n in enumerate(self.lens):
            if n <= 0 or self.new is None:
                continue
            b, o = self.table[i, (n - 1) // self.bs].long(), (n - 1) % self.bs
            for c, e, x in zip(self.kv, self.ex, self.new):
                if self.q8:
                    codes, exps = ref.quantise(x[i])
                    ref.put_rows(c, b, o, codes, self.layout)
                    ref.put_rows(e, b, o, exps, self.layout)
                else:
                    ref.put_rows(c, b, o, x[i], self.layout)

    def expected(self, i):
        """(output, bound) of sequence i from the host caches."""
        n = self.lens[i]
        pos = torch.arange(n)
        pos = pos[ref.visible(n - 1, pos, self.window, self.sinks)]
        k, v = (ref.rows(c, self.table[i], pos, self.bs, self.layout) for c in self.kv)
        if self.q8:
            k, v = (ref.values(x, ref.rows(e, self.table[i], pos, self.bs, self.layout))
                    for x, e in zip((k, v), self.ex))
        o, t = ref.attend(self.q[i:i + 1], k, v, n - 1, pos, self.window, self.sinks, self.scale)
        return o[0], t[0]

    def run(self, dev, out=None, q=None, new=True, **kw):
        k, v, ks, vs = dev
        q = self.q.cuda() if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        nk, nv = (x.cuda() for x in self.new) if self.new and new else (None, None)
        _ops().paged_window_decode(
            out, q, k, v, self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
            scale=self.scale, max_seq_len=kw.pop("max_seq_len", max(max(self.lens), 1)),
            window=self.window, sink_tokens=self.sinks, k_scale=ks, v_scale=vs, new_k=nk,
            new_v=nv, layout=self.layout, **kw)
        return out

    def check(self, out):
        for i, n in enumerate(self.lens):
            if n <= 0:
                assert bool((out[i] == 7).all()), f"row {i} of length {n} was written"
                continue
            o, t = self.expected(i)
            err = (out[i].cpu().double() - o).abs()
            assert bool((err <= t).all()), (
                f"sequence {i} (length {n}): {float((err / t).max())} of the bound")

    def check_caches(self, dev):
        for got, want in zip(dev[:2], self.kv):
            got = got.cpu().view(want.dtype)
            assert torch.equal(got.view(torch.int16 if not self.q8 else torch.uint8),
                               want.view(torch.int16 if not self.q8 else torch.uint8))
        for got, want in zip(dev[2:], self.ex):
            assert want is None or torch.equal(got.cpu(), want)


SHAPES = [(14, 2, 64), (32, 8, 128), (8, 8, 96), (12, 1, 32), (20, 1, 64), (34, 2, 32), (1, 1, 128),
          (16, 1, 128), (24, 2, 96)]
LENS = [1, 2, 15, 16, 17, 0, 31, 100, 33, 257]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("window,sinks,bs,layout", [(0, 0, 16, "hnd"), (40, 4, 16, "nhd"),
                                                    (1, 0, 8, "hnd"), (16, 20, 5, "nhd")])
def test_decode_matches_reference(Hq, Hkv, D, q8, window, sinks, bs, layout):
    c = Case(Hq, Hkv, D, LENS, bs=bs, layout=layout, q8=q8, window=window, sinks=sinks, seed=D + Hq)
    dev = c.device_caches()
    out = c.run(dev)
    assert _ops().check_device_errors() == 0
    c.write_new()
    c.check_caches(dev)
    c.check(out)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens,window,sinks,bs", [
    ([5000], 0, 0, 16), ([5000], 4097, 33, 64), ([20000, 3], 0, 0, 16), ([700] * 3, 1, 1, 1),
    ([3000, 4000], 1000, 5000, 32), ([999], 998, 1, 7), ([1000], 64, 70, 16)])
def test_long_contexts_are_cut_and_merged(lens, window, sinks, bs, q8):
    c = Case(8, 2, 64, lens, bs=bs, q8=q8, window=window, sinks=sinks, seed=len(lens))
    dev = c.device_caches()
    out = c.run(dev)
    again = c.run(dev)
    assert torch.equal(out, again)  # the order of sums does not depend on timing
    assert _ops().check_device_errors() == 0
    c.write_new()
    c.check_caches(dev)
    c.check(out)


def test_larger_max_seq_len_changes_only_the_cut():
    c = Case(32, 8, 128, [300, 40, 1], q8=True, window=0, seed=3)
    out = c.run(c.device_caches(), max_seq_len=100000)
    assert _ops().check_device_errors() == 0
    c.write_new()
    c.check(out)


@pytest.mark.parametrize("q8", [False, True])
def test_fused_write_equals_write_then_decode(q8):
    """The fused call and a separate write followed by the call without new rows agree
    bit for bit."""
    ops = _ops()
    c = Case(32, 8, 128, [64, 65, 1, 900], q8=q8, window=200, sinks=4, seed=8)
    a, b = c.device_caches(), c.device_caches()
    fused = c.run(a)
    slots = torch.tensor([int(c.table[i, (n - 1) // c.bs]) * c.bs + (n - 1) % c.bs
                          for i, n in enumerate(c.lens)], device="cuda")
    new = [x.cuda() for x in c.new]
    if q8:
        ops.kv_quant_write_slots(*b, *new, slots)
    else:
        ops.kv_write_slots(b[0], b[1], *new, slots)
    apart = c.run(b, new=False)
    assert torch.equal(fused, apart)
    for x, y in zip(a, b):
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("q8", [False, True])
def test_views_of_larger_buffers(q8):
    """Q as a plane of a QKV buffer, out with a stride of its own that is no multiple of 8."""
    c = Case(8, 2, 64, [100, 7], q8=q8, window=50, sinks=2, seed=4)
    buf = torch.zeros(2, 12, 64, dtype=torch.float16, device="cuda")
    buf[:, 2:10] = c.q.cuda()
    out = torch.full((2, 9, 67), 7.0, dtype=torch.float16, device="cuda")
    dev = c.device_caches()
    c.run(dev, out=out[:, :8, :64], q=buf[:, 2:10])
    c.write_new()
    c.check(out[:, :8, :64])
    assert bool((out[:, 8] == 7).all()) and bool((out[:, :, 64:] == 7).all())


def test_bad_metadata_is_flagged_and_rows_left_alone():
    ops = _ops()
    from vllm_apple_b200._lib import VA_FLAG_BAD_BLOCK, VA_FLAG_CTX_OVERFLOW
    for lens, splits in (([100, 60, 90], False), ([6000, 5000, 5500], True)):
        c = Case(8, 2, 64, lens, window=0, seed=6, new=False)
        c.table[1, 2] = 10 ** 9
        out = c.run(c.device_caches())
        assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_BAD_BLOCK
        assert bool((out[1] == 7).all())
        c.lens = [lens[0], 0, lens[2]]
        c.check(out)
    # longer than max_seq_len, and longer than the table
    c = Case(8, 2, 64, [100, 60], window=0, seed=6, new=False)
    out = c.run(c.device_caches(), max_seq_len=99)
    assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_CTX_OVERFLOW
    c.lens = [0, 60]
    c.check(out)
    c = Case(8, 2, 64, [100, 60], window=0, seed=6, new=False)
    c.table = c.table[:, :5].contiguous()
    out = c.run(c.device_caches())
    assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_CTX_OVERFLOW
    c.lens = [0, 60]
    c.check(out)


@pytest.mark.parametrize("q8", [False, True])
def test_two_captured_graphs_replay_at_once(q8):
    """Two graphs of cut (workspace-using) calls, captured on one stream and replayed on
    two at the same time, and eager calls between, all give the eager result."""
    cases = [Case(8, 2, 64, [6000, 5000], q8=q8, window=0, seed=s) for s in (1, 2)]
    devs = [c.device_caches() for c in cases]
    want = [c.run(d).clone() for c, d in zip(cases, devs)]
    ins = []
    for c in cases:
        ins.append((c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda(), c.q.cuda(),
                    [x.cuda() for x in c.new], torch.zeros_like(c.q, device="cuda")))

    def call(c, dev, i):
        _ops().paged_window_decode(i[4], i[2], dev[0], dev[1], i[0], i[1], scale=c.scale,
                                   max_seq_len=6000, k_scale=dev[2], v_scale=dev[3],
                                   new_k=i[3][0], new_v=i[3][1])

    graphs = []
    for c, d, i in zip(cases, devs, ins):
        call(c, d, i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c, d, i)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in ins:
        i[4].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[0]):
            extra = cases[1].run(devs[1]) if _ % 7 == 0 else None
    torch.cuda.synchronize()
    for i, w in zip(ins, want):
        assert torch.equal(i[4], w)
    assert extra is None or torch.equal(extra, want[1])


def test_calls_on_a_side_stream():
    c = Case(32, 8, 128, [4000, 10], q8=True, window=0, seed=5)
    dev = c.device_caches()
    want = c.run(dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = c.run(dev)
    s.synchronize()
    assert torch.equal(got, want)
