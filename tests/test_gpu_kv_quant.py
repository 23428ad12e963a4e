"""The e4m3 KV cache: rows quantised by slot and read back, bit for bit against the
64-bit definition."""
import pytest
import torch

import _window_ref as ref

pytestmark = pytest.mark.gpu


def _ops():
    from vllm_apple_b200 import ops
    return ops


def _shape(nb, H, bs, layout):
    return (nb, H, bs) if layout == "hnd" else (nb, bs, H)


def _caches(nb, H, bs, D, layout, seed=0):
    g = torch.Generator().manual_seed(seed)
    s = _shape(nb, H, bs, layout)
    codes = [torch.randint(0, 256, s + (D,), generator=g, dtype=torch.uint8) for _ in range(2)]
    exps = [torch.randint(113, 135, s, generator=g, dtype=torch.uint8) for _ in range(2)]
    return codes, exps


def _f8(t):
    return t.cuda().view(torch.float8_e4m3fn)


def _rows(T, H, D, seed):
    """Rows over the whole range: magnitudes from fp16's smallest to its largest, zeros,
    values half way between two codes, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g)
    x *= torch.exp2(torch.randint(-22, 15, (T, H, 1), generator=g).float())
    x = x.clamp(-65504, 65504).half()
    halves = (torch.arange(D) % 15 + 16.5).half()  # 16.5, 17.5, ...: between codes 16, 17, ...
    if T > 1:
        x[1] = halves
    if T > 2:
        x[2] = 0
    if T > 3:
        x[3, :, 0] = float("inf")
        x[3, :, 1] = float("-inf")
        x[3, :, 2] = float("nan")
    if T > 4:
        x[4, :, D - 1] = 65504
    if T > 5:
        x[5] = 6e-8  # fp16's smallest
    return x


def _assert_codes(got, want, what):
    got = got.cpu().view(torch.uint8)
    nan = (want & 127) == 127
    assert torch.equal((got & 127) == 127, nan), what
    assert torch.equal(got[~nan], want[~nan]), what


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("T,H,D,bs,i64", [
    (1, 1, 32, 16, True), (7, 2, 64, 16, False), (33, 3, 96, 5, True), (257, 8, 128, 16, False),
    (64, 2, 64, 1, True), (40, 1, 128, 64, True), (1500, 5, 96, 8, False), (6, 7, 32, 32, True)])
def test_write_matches_definition(layout, T, H, D, bs, i64):
    ops = _ops()
    nb = T // bs + 3
    codes, exps = _caches(nb, H, bs, D, layout, seed=T)
    k, v = _rows(T, H, D, 1), _rows(T, H, D, 2)
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(3))[:T]
    if T > 8:
        slots[6] = slots[8] = -1
    dk, dv, ks, vs = _f8(codes[0]), _f8(codes[1]), exps[0].cuda(), exps[1].cuda()
    ops.kv_quant_write_slots(dk, dv, ks, vs, k.cuda(), v.cuda(),
                             slots.cuda() if i64 else slots.int().cuda(), layout=layout)
    assert ops.check_device_errors() == 0
    live = slots >= 0
    b, o = slots[live] // bs, slots[live] % bs
    for new, c, e in ((k, codes[0], exps[0]), (v, codes[1], exps[1])):
        qc, qe = ref.quantise(new[live])
        ref.put_rows(c, b, o, qc, layout)
        ref.put_rows(e, b, o, qe, layout)
    _assert_codes(dk, codes[0], "K codes")
    _assert_codes(dv, codes[1], "V codes")
    assert torch.equal(ks.cpu(), exps[0]) and torch.equal(vs.cpu(), exps[1])


def test_write_from_planar_buffer_and_strided_cache():
    """New rows as planes of one QKV buffer, a cache that is a slice of a larger one and
    exponents with a stride of their own."""
    ops = _ops()
    T, H, D, bs, nb = 50, 4, 64, 16, 6
    buf = _rows(T, 3 * H, D, 5)
    dbuf = buf.cuda()
    big = torch.zeros(2, nb, H, bs, 2 * D, dtype=torch.uint8, device="cuda")
    exps = torch.zeros(2, nb, H, bs, 3, dtype=torch.uint8, device="cuda")
    slots = torch.randperm(nb * bs)[:T]
    k, v = big[0, ..., D:].view(torch.float8_e4m3fn), big[1, ..., D:].view(torch.float8_e4m3fn)
    ops.kv_quant_write_slots(k, v, exps[0, ..., 1], exps[1, ..., 1], dbuf[:, H:2 * H],
                             dbuf[:, 2 * H:], slots.cuda())
    want = torch.zeros_like(big, device="cpu")
    wexp = torch.zeros_like(exps, device="cpu")
    for i in range(2):
        c, e = ref.quantise(buf[:, (i + 1) * H:(i + 2) * H])
        want[i, slots // bs, :, slots % bs, D:] = c
        wexp[i, slots // bs, :, slots % bs, 1] = e
    _assert_codes(big, want, "codes")
    assert torch.equal(exps.cpu(), wexp)
    assert ops.check_device_errors() == 0


def test_bad_slots_are_flagged_and_skipped():
    ops = _ops()
    from vllm_apple_b200._lib import VA_FLAG_BAD_SLOT
    codes, exps = _caches(2, 2, 16, 32, "hnd")
    dk, dv, ks, vs = _f8(codes[0]), _f8(codes[1]), exps[0].cuda(), exps[1].cuda()
    rows = torch.randn(3, 2, 32).half().cuda()
    ops.kv_quant_write_slots(dk, dv, ks, vs, rows, rows,
                             torch.tensor([32, -2, 1 << 40], device="cuda"))
    assert ops.check_device_errors(raise_on_error=False) == VA_FLAG_BAD_SLOT
    assert torch.equal(dk.cpu().view(torch.uint8), codes[0])
    assert torch.equal(ks.cpu(), exps[0]) and torch.equal(vs.cpu(), exps[1])
    # an empty call is a no-op
    ops.kv_quant_write_slots(dk, dv, ks, vs, rows[:0], rows[:0],
                             torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert ops.check_device_errors() == 0


@pytest.mark.parametrize("src,dst", [("hnd", "hnd"), ("nhd", "hnd"), ("nhd", "nhd")])
@pytest.mark.parametrize("H,D,bs,lens,renumber", [
    (2, 64, 16, [1, 0, 33, 16, 500], True), (8, 128, 16, [70, 15, 1], False),
    (3, 96, 5, [4, 5, 6, 27], True), (1, 32, 1, [9, 3], False), (5, 128, 64, [64, 65, 200], True),
    (1, 32, 128, [300], True)])
def test_read_back_is_exact(src, dst, H, D, bs, lens, renumber):
    """Every code and every exponent of the range comes back as its value; rows past a
    sequence's end and blocks of no sequence keep what they hold."""
    ops = _ops()
    need = [(n + bs - 1) // bs for n in lens]
    nb = sum(need) + 2
    codes, exps = _caches(nb, H, bs, D, src, seed=D)
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(1)).int()
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    dtable = table.clone()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        dtable[i, :n] = torch.arange(at, at + n)
        at += n
    to = dtable if renumber else table
    want = [torch.full(_shape(nb, H, bs, dst) + (D,), 7.0, dtype=torch.float64) for _ in range(2)]
    for i, n in enumerate(lens):
        pos = torch.arange(n)
        for c, e, w in zip(codes, exps, want):
            val = ref.values(ref.rows(c, table[i], pos, bs, src),
                             ref.rows(e, table[i], pos, bs, src))
            ref.put_rows(w, to[i].long()[pos // bs], pos % bs, val, dst)
    got = [torch.full(w.shape, 7.0, dtype=torch.float16, device="cuda") for w in want]
    ops.kv_dequant_blocks(_f8(codes[0]), _f8(codes[1]), exps[0].cuda(), exps[1].cuda(), *got,
                          table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                          dst_block_table=dtable.cuda() if renumber else None, src_layout=src,
                          dst_layout=dst)
    assert ops.check_device_errors() == 0
    for g, w in zip(got, want):
        assert torch.equal(torch.nan_to_num(g.cpu().double(), nan=12345.0),
                           torch.nan_to_num(w, nan=12345.0))


def test_read_back_flags_bad_blocks_and_long_sequences():
    ops = _ops()
    from vllm_apple_b200._lib import VA_FLAG_BAD_BLOCK, VA_FLAG_CTX_OVERFLOW
    codes, exps = _caches(4, 2, 16, 64, "hnd")
    args = (_f8(codes[0]), _f8(codes[1]), exps[0].cuda(), exps[1].cuda())
    dst = [torch.full((4, 2, 16, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.tensor([[0, 9, 2], [1, 3, 3]], dtype=torch.int32, device="cuda")
    ops.kv_dequant_blocks(*args, *dst, table,
                          torch.tensor([48, 49], dtype=torch.int32, device="cuda"))
    assert (ops.check_device_errors(raise_on_error=False)
            == VA_FLAG_BAD_BLOCK | VA_FLAG_CTX_OVERFLOW)
    for d, c, e in zip(dst, codes, exps):
        v = ref.values(c, e)
        for b in (0, 2):  # the blocks around the bad one are read
            assert torch.equal(torch.nan_to_num(d[b].cpu().double()), torch.nan_to_num(v[b]))
        assert bool((d[1] == 7).all()) and bool((d[3] == 7).all())


def test_round_trip_error_is_half_a_step():
    """Written and read back, a value in a row's normal range is off by at most 2^-4 of
    itself (half an e4m3 step), a smaller one by half the smallest step 2^-10 2^e."""
    ops = _ops()
    T, H, D, bs = 200, 4, 128, 16
    nb = T // bs + 1
    x = torch.randn(T, H, D).half()
    k = torch.zeros(nb, H, bs, D, dtype=torch.float8_e4m3fn, device="cuda")
    v, ks = torch.zeros_like(k), torch.zeros(nb, H, bs, dtype=torch.uint8, device="cuda")
    vs = torch.zeros_like(ks)
    ops.kv_quant_write_slots(k, v, ks, vs, x.cuda(), x.cuda(), torch.arange(T, device="cuda"))
    dk, dv = (torch.zeros(nb, H, bs, D, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.arange(nb, dtype=torch.int32, device="cuda")[None]
    ops.kv_dequant_blocks(k, v, ks, vs, dk, dv, table,
                          torch.tensor([T], dtype=torch.int32, device="cuda"))
    back = dk.cpu().permute(0, 2, 1, 3).reshape(-1, H, D)[:T].double()
    a = x.double().abs().amax(-1, keepdim=True)
    step = 2.0 ** -10 * 2 * a / 448  # 2^e < 2 a / 448
    err = (back - x.double()).abs()
    assert bool((err <= torch.maximum(x.double().abs() * 2.0 ** -4, step)).all())
    assert torch.equal(dk, dv)
