"""Prompt chunks whose scores rise from key tile to key tile, so that a row's reference
maximum moves and its sums so far are rescaled, for some rows of a warp and not for others;
and rises that stay below the bound of 2^12 at which it moves."""
import math

import pytest
import torch

import _window_ref as ref
from test_gpu_window_prefill import Case

pytestmark = pytest.mark.gpu

KEYS, BOUND = 128, 12.0  # keys of a tile; log2 of what a power may reach before a move


def _make(D, q8, levels, window, sinks, bs):
    """Three chunks of G = 4; the log2 score of a rising row (two of three) lies near
    levels[t] in key tile t, and V is scaled so that every tile within 2^15 of the last one
    counts in the result."""
    c = Case(8, 2, D, [(0, 300), (400, 120), (630, 2)], bs=bs, q8=q8, window=window, sinks=sinks,
             seed=D + len(levels))
    g = torch.Generator().manual_seed(5)
    c.q *= 0.05
    c.q[:, :, 0] = (torch.rand(c.q.shape[:2], generator=g) < 0.67).half()
    for i, n in enumerate(c.lens):
        for p in range(n):
            b, o = int(c.table[i, p // bs]), p % bs
            if b < 0:
                continue  # no query sees it
            t = min(p // KEYS, len(levels) - 1)
            k, v = (torch.randn(2, D, generator=g) for _ in range(2))
            k[:, 0] = levels[t] / (c.scale * math.log2(math.e))
            v *= 2.0 ** min(max(levels[-1] - levels[t], 0), 12)
            for x, cache, ex in zip((k.half(), v.half()), c.kv, c.ex):
                if q8:
                    codes, e = ref.quantise(x)
                    ref.put_rows(cache, b, o, codes, c.layout)
                    ref.put_rows(ex, b, o, e, c.layout)
                else:
                    ref.put_rows(cache, b, o, x, c.layout)
    return c


def _moves(c, i):
    """Per (token, head) of sequence i: rises of the tiles' maxima over the reference maximum
    at which it moves, and those at which it stays (the largest of each, 0: none)."""
    first, n = c.chunks[i][0], c.lens[i]
    pos = torch.arange(n)
    p = first + torch.arange(n - first)
    see = ref.visible(p[:, None], pos[None], c.window, c.sinks)
    pos = pos[see.any(0)]
    k = c.cache_rows(i, pos)[0].double().repeat_interleave(4, 1)
    q = c.q[c.start[i]:c.start[i + 1]].double()
    s = torch.einsum("nhd,mhd->nhm", q, k) * c.scale * math.log2(math.e)
    s = torch.where(see[:, pos][:, None], s, -math.inf)
    m = torch.full(s.shape[:2], -math.inf, dtype=torch.float64)
    moved, stayed = torch.zeros_like(m), torch.zeros_like(m)
    for t in range((n + KEYS - 1) // KEYS):
        cols = pos // KEYS == t
        if not bool(cols.any()):
            continue
        top = s[..., cols].amax(-1)
        rise = torch.where(torch.isfinite(m) & torch.isfinite(top), top - m, 0.0)
        go = rise > BOUND
        moved = torch.maximum(moved, torch.where(go, rise, 0.0))
        stayed = torch.maximum(stayed, torch.where(go, 0.0, rise))
        m = torch.where(go | ~torch.isfinite(m), torch.maximum(m, top), m)
    return moved, stayed


# (levels by key tile, window, sinks, range of the largest move of sequence 1, of its largest stay);
# e4m3 keys move a level by up to 2^-4 of it
RISES = [
    ((0, 12.8), 0, 0, (12, 14), (0, 1)),
    ((0, 11.2), 0, 0, (0, 0), (10, 12)),
    ((0, 11.2, 12.9, 24), 0, 0, (12, 14), (10, 12)),
    ((0, 40, 40, 80), 0, 0, (37, 43), (0, 1)),
    ((4, 0, -3, 9, 22), 0, 0, (16, 20), (4, 6)),
    ((0, 3, 14, 20, 33), 200, 4, (17, 21), (4, 7)),
]


@pytest.mark.parametrize("bs", [16, 24])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("levels,window,sinks,moves,stays", RISES)
def test_reference_maximum_moves(levels, window, sinks, moves, stays, D, q8, bs):
    from vllm_apple_b200 import ops
    c = _make(D, q8, levels, window, sinks, bs)
    moved, stayed = _moves(c, 1)
    assert moves[0] <= float(moved.max()) <= moves[1]
    assert stays[0] <= float(stayed.max()) <= stays[1]
    if moves[1]:  # rows of one warp (8 tokens of 4 heads) that move and rows that do not
        warps = (moved[:, :4] > 0).reshape(-1, 32)
        assert bool((warps.any(1) & ~warps.all(1)).any())
    out = c.run()
    assert torch.equal(out, c.run())
    assert ops.check_device_errors() == 0
    c.check(out)
