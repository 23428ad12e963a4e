"""64-bit plain forms of the e4m3 KV cache and of windowed attention, with error bounds."""
import math

import torch

F64 = torch.float64


def e4m3_values():
    """Value of every e4m3 code (sign, 4 exponent bits with bias 7, 3 fraction bits)."""
    t = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        v = math.nan if c & 127 == 127 else v
        t.append(-v if c & 128 else v)
    return torch.tensor(t, dtype=F64)


def quantise(x):
    """(codes uint8, exponent bytes uint8) of rows x [..., D], by search among the values."""
    x = x.to(F64)
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    e = torch.full(a.shape, -14, dtype=torch.int64)
    for k in range(-14, 7):
        e += (a > 448.0 * 2.0 ** k).long()
    p2 = torch.tensor([2.0 ** k for k in range(-14, 8)], dtype=F64)[e + 14]
    y = (x / p2[..., None]).clamp(-448, 448)
    pos = e4m3_values()[:127].contiguous()
    m = torch.nan_to_num(y).abs().contiguous()
    hi = torch.searchsorted(pos, m).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dh, dl = pos[hi] - m, m - pos[lo]
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = torch.where(torch.isnan(x), 127, code + 128 * torch.signbit(y).long())
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def values(codes, exps):
    """64-bit values of quantised rows."""
    p2 = torch.tensor([2.0 ** (k - 127) for k in range(256)], dtype=F64)[exps.long()]
    return e4m3_values()[codes.long()] * p2[..., None]


def rows(cache, table_row, pos, bs, layout):
    """Rows [len(pos), H, ...] of a cache (or its exponents) at positions ``pos``."""
    b, o = table_row.long()[pos // bs], pos % bs
    return cache[b, o] if layout == "nhd" else cache[b, :, o]


def put_rows(cache, block, off, new, layout):
    if layout == "nhd":
        cache[block, off] = new
    else:
        cache[block, :, off] = new


def visible(p, j, window, sinks):
    """Whether the query at p sees key j (broadcast)."""
    see = j <= p
    if window > 0:
        see = see & ((p - j < window) | (j < sinks))
    return see


def attend(q, k, v, first, pos, window, sinks, scale):
    """64-bit output and bound of queries q [n, Hq, D] at positions first.. over the keys
    k, v [m, Hkv, D] at positions ``pos`` [m].

    The bound adds, per output value o = sum p v / sum p with A = sum p |v| / sum p:
      * the result's rounding to fp16: 2^-11 |o| (2^-25 where it is subnormal);
      * P rounded to fp16 before the second product: 2^-11 per weight, so 2^-11 A, and
        2^-25 per weight below fp16's normal range, so 2^-25 sum |v| / sum p;
      * fp32 sums: a score of D products is off by (D + 2) 2^-24 sum |q_i k_i| scale, which
        moves a weight by twice that (the maximum moves too), and so o by twice that again
        (weights and their sum); the sums over m keys by m 2^-24; the power of two by 2^-21
        (its own error and its argument's rounding).
    """
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    see = visible((first + torch.arange(n))[:, None], pos[None, :], window, sinks)
    seen = see.any(0)
    k, v, see = k[seen], v[seen], see[:, seen]
    ke, ve = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("nhd,mhd->nhm", q, ke) * scale
    mag = torch.einsum("nhd,mhd->nhm", q.abs(), ke.abs()) * scale
    s = torch.where(see[:, None], s, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    tot = e.sum(-1)[..., None]
    o = torch.einsum("nhm,mhd->nhd", torch.where(see[:, None], e, 0.0), ve) / tot
    A = torch.einsum("nhm,mhd->nhd", e, ve.abs()) / tot
    V = torch.einsum("nhm,mhd->nhd", see[:, None].to(F64).expand_as(e), ve.abs()) / tot
    ds = (D + 2) * 2.0 ** -24 * torch.where(see[:, None], mag, 0.0).amax(-1)[..., None]
    bound = (2.0 ** -11 * (o.abs() + A) + 2.0 ** -25 * (1 + V)
             + A * (4 * ds + 2 * k.shape[0] * 2.0 ** -24 + 2 * 2.0 ** -21))
    return o, bound
