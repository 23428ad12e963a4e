"""Visible keys whose score is -inf (an infinity in an fp16 K row): their weight is 0, and a
row with any other visible key stays finite, however the keys fall to tiles, warps and CTAs."""
import math

import pytest
import torch

import _window_ref as ref
from test_gpu_window_decode import Case

pytestmark = pytest.mark.gpu


def _make(Hq, Hkv, D, n, infinite, new, **kw):
    """A sequence of n keys; K rows at the positions ``infinite`` score -inf for every head."""
    c = Case(Hq, Hkv, D, [n, 50], new=new, seed=n, **kw)
    c.q[:, :, 0] = c.q[:, :, 0].abs() + 0.5
    for p in infinite:
        if new and p == n - 1:
            c.new[0][0, :, 0] = -math.inf
            continue
        b, o = c.table[0, p // c.bs].long(), p % c.bs
        row = ref.rows(c.kv[0], c.table[0], torch.tensor([p]), c.bs, c.layout)[0].clone()
        row[:, 0] = -math.inf
        ref.put_rows(c.kv[0], b, o, row, c.layout)
    return c


def _expected(c, infinite):
    """64-bit output and bound of sequence 0: a weight of 0 takes no part."""
    n = c.lens[0]
    pos = torch.arange(n)
    keep = ref.visible(n - 1, pos, c.window, c.sinks)
    keep[list(infinite)] = False
    pos = pos[keep]
    k, v = (ref.rows(x, c.table[0], pos, c.bs, c.layout) for x in c.kv)
    o, t = ref.attend(c.q[:1], k, v, n - 1, pos, c.window, c.sinks, c.scale)
    return o[0], t[0]


CASES = [
    (17, {16}, 0, 0),                               # the newest key alone in its tile
    (33, set(range(16)), 0, 0),                     # a warp's only tile
    (200, set(range(16)) | set(range(64, 80)), 0, 0),   # a warp's first two tiles
    (161, {160}, 40, 4),
    (161, {0, 1, 2, 3}, 40, 4),                     # the sinks
    (49, set(range(48)), 0, 0),                     # everything but the newest
    (6001, {6000}, 0, 0),                           # cut over several CTAs
    (6001, set(range(1000, 6000)), 0, 0),           # whole ranges
]


@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (32, 8, 128), (16, 1, 96)])
@pytest.mark.parametrize("n,infinite,window,sinks", CASES)
def test_keys_of_weight_zero(n, infinite, window, sinks, Hq, Hkv, D, new):
    from vllm_apple_b200 import ops
    c = _make(Hq, Hkv, D, n, infinite, new, window=window, sinks=sinks)
    out = c.run(c.device_caches())
    assert ops.check_device_errors() == 0
    c.write_new()
    o, t = _expected(c, infinite)
    assert bool(((out[0].cpu().double() - o).abs() <= t).all())
    o, t = c.expected(1)
    assert bool(((out[1].cpu().double() - o).abs() <= t).all())
    # the same rows as chunks of one token
    kv = [x.cuda() for x in c.kv]
    chunk = torch.full_like(c.q, 7.0, device="cuda")
    ops.paged_window_prefill(chunk, c.q.cuda(), *kv, c.table.cuda(),
                             torch.tensor([0, 1, 2], dtype=torch.int32).cuda(),
                             torch.tensor(c.lens, dtype=torch.int32).cuda(), scale=c.scale,
                             window=window, sink_tokens=sinks)
    assert ops.check_device_errors() == 0
    o, t = _expected(c, infinite)
    assert bool(((chunk[0].cpu().double() - o).abs() <= t).all())


@pytest.mark.parametrize("n", [17, 6001])
def test_rows_without_any_finite_score_are_nan(n):
    c = _make(8, 2, 64, n, set(range(n)), False, window=0)
    out = c.run(c.device_caches())
    assert bool(torch.isnan(out[0]).all())
    o, t = c.expected(1)
    assert bool(((out[1].cpu().double() - o).abs() <= t).all())
