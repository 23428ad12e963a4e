"""Measured cases of the 8-bit KV cache and of windowed attention over paged caches.

Four operators, each in its plain form (elementary torch operations in 32 bits)
and, where ``own`` is true, as the call a user makes of ``vllm_apple_b200.ops``:

  write    new K/V rows quantised to e4m3 with one power-of-two exponent per
           (token, kv head) and scattered into a paged cache by slot
  read     the active blocks of an e4m3 cache read back into an fp16 cache
  decode   one new token per sequence: attention over its visible keys in an
           fp16 or e4m3 paged cache, with the write of the new row
  prefill  a chunk of new tokens per sequence: causal attention over the visible
           keys in an fp16 or e4m3 paged cache that already holds them

A query at position p sees the keys j <= p with p - j < window (window 0: all of
them) or j < sinks.  An e4m3 row of D values holds codes c and one exponent e and
stands for c * 2^e, with e = ceil(log2(max|x| / 448)) clamped to [-14, 7].
"""
import math
import os
import random
import sys

import torch

own = False

# Shapes (query heads, kv heads, head size) of the repository's two configurations.
SMALL = {"hq": 14, "hkv": 2, "d": 64}
LARGE = {"hq": 32, "hkv": 8, "d": 128}


def listed():
    return [
        # one step's new rows of 64 sequences: a handful of kilobytes, launch latency only
        dict(SMALL, name="write_64_rows", op="write", tokens=64, pad=0, bs=16, nhd=False, shape=1),
        # the new rows of long prompts, with the padding rows a fixed-size batch carries
        dict(LARGE, name="write_16384_padded", op="write", tokens=16384, pad=301, bs=16, nhd=True,
             shape=2),
        # four half-filled contexts handed to a consumer that reads fp16
        dict(LARGE, name="read_4_contexts", op="read", seqs=4, lo=1, hi=4096, bs=16, nhd=False,
             renumber=True, shape=3),
        # a whole serving batch moved out of the 8-bit cache
        dict(LARGE, name="read_64_contexts", op="read", seqs=64, lo=512, hi=8192, bs=16, nhd=True,
             renumber=False, shape=4),
        # the smallest step: 4 sequences, a short window, fp16
        dict(SMALL, name="decode_4_window_128", op="decode", seqs=4, lo=32, hi=512, bs=16,
             nhd=False, q8=False, window=128, sinks=4, write=True, shape=5),
        # a middle batch of ragged contexts, the whole context in 8 bits
        dict(SMALL, name="decode_64_q8", op="decode", seqs=64, lo=1, hi=4096, bs=16, nhd=False,
             q8=True, window=0, sinks=0, write=True, shape=6),
        # a serving batch whose layers see 1024 tokens and the first 4
        dict(LARGE, name="decode_128_window_1024", op="decode", seqs=128, lo=512, hi=8192, bs=16,
             nhd=True, q8=False, window=1024, sinks=4, write=True, shape=7),
        # the same batch with all of its context, in 8 bits
        dict(LARGE, name="decode_128_q8", op="decode", seqs=128, lo=512, hi=8192, bs=16, nhd=False,
             q8=True, window=0, sinks=0, write=True, shape=8),
        # one user's very long document: one row of work per kv head, split over the context
        dict(LARGE, name="decode_1_long_q8", op="decode", seqs=1, lo=131000, hi=131000, bs=16,
             nhd=False, q8=True, window=0, sinks=0, write=True, shape=9),
        # short ragged questions after a prefix, in 8 bits
        dict(SMALL, name="prefill_ragged_q8", op="prefill", seqs=7, chunk_lo=1, chunk_hi=100, lo=0,
             hi=600, bs=16, nhd=False, q8=True, window=256, sinks=3, shape=10),
        # one chunked-prefill step: 4 chunks of 512 with prior context, a window and sinks
        dict(LARGE, name="prefill_4x512_window_1024", op="prefill", seqs=4, chunk_lo=512,
             chunk_hi=512, lo=0, hi=4096, bs=16, nhd=False, q8=False, window=1024, sinks=4,
             shape=11),
        # a long prompt in one piece under a 4096-token window, cache in 8 bits
        dict(LARGE, name="prefill_8192_window_4096_q8", op="prefill", seqs=1, chunk_lo=8192,
             chunk_hi=8192, lo=0, hi=0, bs=16, nhd=True, q8=True, window=4096, sinks=4, shape=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    hq, hkv, d = rng.choice([(14, 2, 64), (32, 8, 128), (8, 8, 96), (12, 1, 32), (24, 2, 128),
                             (16, 4, 64), (5, 5, 128), (40, 8, 128)])
    c = dict(hq=hq, hkv=hkv, d=d, bs=rng.choice([8, 16, 16, 32, 64]), nhd=rng.random() < 0.5,
             shape=rng.randrange(1 << 30))
    c["op"] = rng.choice(["write", "read", "decode", "decode", "prefill", "prefill"])
    if c["op"] == "write":
        c.update(tokens=_log_int(rng, 1, 16000), pad=rng.choice([0, 0, 1, 37]))
        return c
    if c["op"] == "read":
        hi = _log_int(rng, 1, 8192)
        c.update(seqs=_log_int(rng, 1, 48), lo=1, hi=hi, renumber=rng.random() < 0.5)
        return c
    c.update(q8=rng.random() < 0.5, window=rng.choice([0, 1, _log_int(rng, 2, 6000)]),
             sinks=rng.choice([0, 1, 4, 4, rng.randrange(2, 70)]))
    if c["op"] == "decode":
        seqs = _log_int(rng, 1, 160)
        hi = _log_int(rng, 1, min(100000, 300000 // seqs))
        c.update(seqs=seqs, lo=1, hi=hi, write=rng.random() < 0.8)
        return c
    seqs = _log_int(rng, 1, 12)
    chunk = _log_int(rng, 1, max(1, 4096 // seqs))
    c.update(seqs=seqs, chunk_lo=max(1, chunk // 2), chunk_hi=chunk, lo=0,
             hi=_log_int(rng, 1, 2800))
    return c


# ---------------------------------------------------------------------------
# sizes of a case (plain integers; the values depend on the seed, these do not)
# ---------------------------------------------------------------------------
def _sizes(case):
    """(context lengths, new-token counts) of the case's sequences."""
    r = random.Random(case["shape"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    if case["op"] != "prefill":
        return lens, [1] * len(lens)
    new = [r.randint(case["chunk_lo"], case["chunk_hi"]) for _ in lens]
    return [a + b for a, b in zip(lens, new)], new


def _visible_pairs(first, last, window, sinks):
    """Sum over positions p in [first, last] of the number of keys p sees."""
    if window <= 0:
        return (last * (last + 1) - first * (first - 1)) // 2 + (last - first + 1)
    total = 0
    for p in range(first, last + 1):
        lo = max(0, p - window + 1)
        total += p + 1 - lo + min(sinks, lo)
    return total


def _seen_keys(first, last, window, sinks):
    """Keys that at least one of the positions [first, last] sees."""
    lo = max(0, first - window + 1) if window > 0 else 0
    return last + 1 - lo + min(sinks, lo)


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        n = case["tokens"]
        return {"bytes": n * hkv * (2 * d * 2 + 2 * d + 2) + n * 8, "flops": 0}
    lens, new = _sizes(case)
    pages = sum((n + case["bs"] - 1) // case["bs"] for n in lens)
    if case["op"] == "read":
        n = sum(lens)
        return {"bytes": n * hkv * (2 * d + 2 + 2 * d * 2) + pages * 4, "flops": 0}
    row = 2 * d + 2 if case["q8"] else 4 * d
    seen = sum(_seen_keys(n - m, n - 1, case["window"], case["sinks"])
               for n, m in zip(lens, new))
    pairs = sum(_visible_pairs(n - m, n - 1, case["window"], case["sinks"])
                for n, m in zip(lens, new))
    moved = seen * hkv * row + sum(new) * hq * d * 4 + (seen // case["bs"] + len(lens)) * 4
    if case.get("write"):
        moved += len(lens) * hkv * (4 * d + (row if case["q8"] else 0))
    return {"bytes": moved, "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _fill_codes(shape, g):
    """Random e4m3 codes as a quantised row holds them (no NaN code)."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    return (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _cache(case, blocks, q8, g):
    """K and V caches (and their exponents) of ``blocks`` blocks in the case's layout."""
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    rows = (blocks, bs, hkv) if case["nhd"] else (blocks, hkv, bs)
    if not q8:
        kv = [torch.randn(rows + (d,), generator=g, device="cuda", dtype=torch.float16)
              for _ in range(2)]
        return kv + [None, None]
    kv = [_fill_codes(rows + (d,), g) for _ in range(2)]
    # rows of unit-variance values have exponents near log2(3 / 448)
    ex = [torch.randint(118, 122, rows, generator=g, device="cuda", dtype=torch.uint8)
          for _ in range(2)]
    return kv + ex


def _tables(lens, bs, gen, device="cuda"):
    need = [(n + bs - 1) // bs for n in lens]
    blocks = sum(need) + 3
    perm = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table.to(device), blocks


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    s = {"case": case, "layout": "nhd" if case["nhd"] else "hnd"}

    def rows(n, heads):
        return torch.randn((n, heads, d), generator=g, device="cuda", dtype=torch.float16)

    if case["op"] == "write":
        n = case["tokens"]
        blocks = (n + bs - 1) // bs + 2
        s["k"], s["v"], s["ks"], s["vs"] = _cache(case, blocks, True, g)
        slots = torch.randperm(blocks * bs, generator=gen)[:n + case["pad"]]
        slots = torch.cat([slots[:n], torch.full((case["pad"],), -1, dtype=torch.int64)])
        s["slots"] = slots[torch.randperm(len(slots), generator=gen)].cuda()
        s["new_k"], s["new_v"] = rows(len(slots), hkv), rows(len(slots), hkv)
        # values as activations have them: some channels much larger than the rest
        s["new_k"][:, :, ::17] *= 12
        return s
    lens, new = _sizes(case)
    s["lens"], s["new"] = lens, new
    s["table"], blocks = _tables(lens, bs, gen)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    if case["op"] == "read":
        s["k"], s["v"], s["ks"], s["vs"] = _cache(case, blocks, True, g)
        s["dk"], s["dv"] = (torch.zeros(s["k"].shape, dtype=torch.float16, device="cuda")
                            for _ in range(2))
        s["dtable"] = None
        if case["renumber"]:  # consecutive blocks in the destination
            live = s["table"] >= 0
            s["dtable"] = torch.where(live, (torch.cumsum(live.reshape(-1), 0) - 1)
                                      .reshape(live.shape), -1).to(torch.int32)
        return s
    s["k"], s["v"], s["ks"], s["vs"] = _cache(case, blocks, case["q8"], g)
    s["scale"] = 1.0 / math.sqrt(d)
    s["q"] = rows(sum(new), hq)
    s["out"] = torch.zeros_like(s["q"])
    s["max_len"] = max(lens)
    if case["op"] == "decode":
        s["new_k"] = rows(len(lens), hkv) if case["write"] else None
        s["new_v"] = rows(len(lens), hkv) if case["write"] else None
    else:
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        s["start"] = start
        s["qsl"] = torch.tensor(start, dtype=torch.int32).cuda()
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _quantise(x):
    """(codes, exponent bytes) of rows x [..., D]."""
    x = x.float()
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(a > 0, e - 9 + (m > 0.875), -14).clamp(-14, 7)
    y = (x * _power(-e)[..., None]).clamp(-448.0, 448.0)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _power(e):
    """fp32 2^e for integers e, from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _values(codes, exponents):
    return codes.float() * _power(exponents.to(torch.int32) - 127)[..., None]


def _at(case, block, off):
    """Index of the rows (block, off) of every head in a cache of the case's layout."""
    return (block, off) if case["nhd"] else (block, slice(None), off)


def _store(s, block, off, new_k, new_v):
    """Write rows [n, heads, D] at (block, off) of the state's caches."""
    at = _at(s["case"], block, off)
    for cache, ex, new in ((s["k"], s["ks"], new_k), (s["v"], s["vs"], new_v)):
        if ex is None:
            cache[at] = new
        else:
            codes, exps = _quantise(new)
            cache.view(torch.uint8)[at] = codes.view(torch.uint8)
            ex[at] = exps


def _gather(s, i, pos):
    """fp32 K and V [heads, keys, D] of sequence i at the positions ``pos``."""
    case = s["case"]
    block, off = s["table"][i][pos // case["bs"]].long(), pos % case["bs"]
    at = _at(case, block, off)
    got = []
    for cache, ex in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        x = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn) if ex is not None else cache[at]
        x = x.float() if ex is None else _values(x, ex[at])
        got.append(x.transpose(0, 1))
    return got


def _attend(s, i, q, first):
    """fp16 output [n, hq, D] of queries q [n, hq, D] of sequence i at positions first..first+n-1."""
    case = s["case"]
    n, hq, d = q.shape
    w, sinks = case["window"], case["sinks"]
    last = first + n - 1
    lo = max(0, first - w + 1) if w > 0 else 0
    pos = torch.arange(lo, last + 1, device="cuda")
    if lo > 0 and sinks > 0:
        pos = torch.cat([torch.arange(min(sinks, lo), device="cuda"), pos])
    k, v = _gather(s, i, pos)
    hkv = k.shape[0]
    qq = q.float().reshape(n, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
    sc = torch.matmul(qq, k.transpose(1, 2)) * s["scale"]
    p = first + torch.arange(n, device="cuda")[:, None]
    see = pos[None, :] <= p
    if w > 0:
        see = see & ((p - pos[None, :] < w) | (pos[None, :] < sinks))
    sc = sc.reshape(hkv, hq // hkv, n, -1).masked_fill(~see, float("-inf"))
    sc = torch.exp(sc - sc.amax(-1, keepdim=True))
    sc = sc / sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.reshape(hkv, -1, sc.shape[-1]), v)
    return o.reshape(hkv, hq // hkv, n, d).permute(2, 0, 1, 3).reshape(n, hq, d).half()


def _plain(s):
    case = s["case"]
    bs = case["bs"]
    if case["op"] == "write":
        live = s["slots"] >= 0
        slots = s["slots"][live]
        _store(s, slots // bs, slots % bs, s["new_k"][live], s["new_v"][live])
        return {"k": s["k"], "v": s["v"], "k_exp": s["ks"], "v_exp": s["vs"]}
    if case["op"] == "read":
        for i, n in enumerate(s["lens"]):
            pos = torch.arange(n, device="cuda")
            k, v = _gather(s, i, pos)
            table = s["table"] if s["dtable"] is None else s["dtable"]
            at = _at(case, table[i][pos // bs].long(), pos % bs)
            s["dk"][at] = k.transpose(0, 1).half()
            s["dv"][at] = v.transpose(0, 1).half()
        return {"k": s["dk"], "v": s["dv"]}
    if case["op"] == "decode":
        if case["write"]:
            p = (s["seq_lens"] - 1).long()
            block = s["table"].gather(1, (p // bs)[:, None])[:, 0].long()
            _store(s, block, p % bs, s["new_k"], s["new_v"])
        for i, n in enumerate(s["lens"]):
            s["out"][i:i + 1] = _attend(s, i, s["q"][i:i + 1], n - 1)
        return _decode_outputs(s)
    step = 512  # query rows at a time: bounds the scores held at once
    for i, n in enumerate(s["lens"]):
        a, b = s["start"][i], s["start"][i + 1]
        for t in range(a, b, step):
            u = min(t + step, b)
            s["out"][t:u] = _attend(s, i, s["q"][t:u], n - (b - a) + (t - a))
    return {"out": s["out"]}


def _decode_outputs(s):
    r = {"out": s["out"]}
    if s["case"]["write"]:
        r.update(k=s["k"], v=s["v"])
        if s["ks"] is not None:
            r.update(k_exp=s["ks"], v_exp=s["vs"])
    return r


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _ops():
    path = os.path.join(os.getcwd(), "vllm-apple_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vllm_apple_b200 import ops
    return ops


def _own(s):
    ops = _ops()
    case, layout = s["case"], s["layout"]
    if case["op"] == "write":
        ops.kv_quant_write_slots(s["k"], s["v"], s["ks"], s["vs"], s["new_k"], s["new_v"],
                                 s["slots"], layout=layout)
        return {"k": s["k"], "v": s["v"], "k_exp": s["ks"], "v_exp": s["vs"]}
    if case["op"] == "read":
        ops.kv_dequant_blocks(s["k"], s["v"], s["ks"], s["vs"], s["dk"], s["dv"], s["table"],
                              s["seq_lens"], dst_block_table=s["dtable"], src_layout=layout,
                              dst_layout=layout)
        return {"k": s["dk"], "v": s["dv"]}
    if case["op"] == "decode":
        ops.paged_window_decode(s["out"], s["q"], s["k"], s["v"], s["table"], s["seq_lens"],
                                scale=s["scale"], max_seq_len=s["max_len"],
                                window=case["window"], sink_tokens=case["sinks"],
                                k_scale=s["ks"], v_scale=s["vs"], new_k=s["new_k"],
                                new_v=s["new_v"], layout=layout)
        return _decode_outputs(s)
    ops.paged_window_prefill(s["out"], s["q"], s["k"], s["v"], s["table"], s["qsl"],
                             s["seq_lens"], scale=s["scale"], window=case["window"],
                             sink_tokens=case["sinks"], k_scale=s["ks"], v_scale=s["vs"],
                             layout=layout)
    return {"out": s["out"]}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _e4m3_table():
    """Value of every e4m3 code: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f is NaN."""
    t = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        v = float("nan") if c & 127 == 127 else v
        t.append(-v if c & 128 else v)
    return torch.tensor(t, dtype=torch.float64, device="cuda")


def _two_to(e):
    """64-bit 2^e for integers e in [-127, 128], by table: a device pow() need not be exact."""
    t = torch.tensor([2.0 ** k for k in range(-127, 129)], dtype=torch.float64, device="cuda")
    return t[e.long() + 127]


def _exact_rows(x):
    """(e4m3 value, exponent) of rows by search among the e4m3 values, ties to the even code."""
    x = x.double()
    a = x.abs().amax(-1)
    e = torch.full(a.shape, -14, dtype=torch.int64, device="cuda")
    for k in range(-14, 7):  # the smallest exponent whose 448 2^e reaches a, at most 7
        e += (a > 448.0 * 2.0 ** k).long()
    y = (x / _two_to(e)[..., None]).clamp(-448, 448)
    pos = _e4m3_table()[:127]
    m = y.abs()
    hi = torch.searchsorted(pos, m.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dh, dl = pos[hi] - m, m - pos[lo]
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(pos[code], y), e + 127


def _exact_cache(s):
    """The state's caches as 64-bit values [blocks, bs, heads, D], and exponents (or None)."""
    out = []
    table = _e4m3_table()
    for name, ex in (("k", "ks"), ("v", "vs")):
        x = s[name]
        if s[ex] is None:
            x = x.double()
        else:
            x = table[x.view(torch.uint8).long()]
        out.append((x, None if s[ex] is None else s[ex].long()))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    nhd, bs = case["nhd"], case["bs"]

    def put(dst, block, off, row):
        if nhd:
            dst[block, off] = row
        else:
            dst[block, :, off] = row

    if case["op"] == "write":
        (k, ke), (v, ve) = _exact_cache(s)
        live = (s["slots"] >= 0).nonzero()[:, 0]
        sl = s["slots"][live]
        for cache, ex, new in ((k, ke, s["new_k"]), (v, ve, s["new_v"])):
            val, e = _exact_rows(new[live])
            put(cache, sl // bs, sl % bs, val)
            put(ex, sl // bs, sl % bs, e)
        return {"k": k, "v": v, "k_exp": ke, "v_exp": ve}
    table = _e4m3_table()

    def rows(name, ex, i, n, sel=None):
        """64-bit values [n, heads, D] of the first n positions of sequence i (or of ``sel``)."""
        p = torch.arange(n, device="cuda") if sel is None else sel
        b, o = s["table"][i].long()[torch.div(p, bs, rounding_mode="floor")], torch.remainder(p, bs)
        raw = s[name] if s[ex] is None else s[name].view(torch.uint8)
        x = raw[b, o] if nhd else raw[b, :, o]
        if s[ex] is None:
            return x.double()
        e = s[ex][b, o] if nhd else s[ex][b, :, o]
        return table[x.long()] * _two_to(e.long() - 127)[..., None]

    lens, new = s["lens"], s["new"]
    if case["op"] == "read":
        if sum(lens) * case["hkv"] * case["d"] > 1 << 28:
            return None
        dk, dv = s["dk"].double(), s["dv"].double()
        dst = s["table"] if s["dtable"] is None else s["dtable"]
        for i, n in enumerate(lens):
            p = torch.arange(n, device="cuda")
            b, o = dst[i].long()[torch.div(p, bs, rounding_mode="floor")], torch.remainder(p, bs)
            put(dk, b, o, rows("k", "ks", i, n))
            put(dv, b, o, rows("v", "vs", i, n))
        return {"k": dk, "v": dv}
    result = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    if case["op"] == "decode" and case["write"]:
        p = (s["seq_lens"] - 1).long()
        b = s["table"][torch.arange(len(lens), device="cuda"), p // bs].long()
        (k, ke), (v, ve) = _exact_cache(s)
        for cache, ex, nw, name, en in ((k, ke, s["new_k"], "k", "ks"),
                                        (v, ve, s["new_v"], "v", "vs")):
            if ex is None:
                put(cache, b, p % bs, nw.double())
                put(s[name], b, p % bs, nw)
            else:
                val, e = _exact_rows(nw)
                put(cache, b, p % bs, val)
                put(ex, b, p % bs, e)
                put(s[name].view(torch.uint8), b, p % bs,
                    val.to(torch.float8_e4m3fn).view(torch.uint8))
                put(s[en], b, p % bs, e.to(torch.uint8))
        result.update(k=k, v=v)
        if ke is not None:
            result.update(k_exp=ke, v_exp=ve)
    hq, hkv = case["hq"], case["hkv"]
    at = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        for c in range(0, m, 256):
            t = torch.arange(n - m + c, min(n - m + c + 256, n), device="cuda")
            j = torch.arange(n, device="cuda")
            keep = j[None, :] <= t[:, None]
            if case["window"] > 0:
                keep &= (t[:, None] - j[None, :] < case["window"]) | (j < case["sinks"])[None, :]
            some = keep.any(0).nonzero()[:, 0]
            keep = keep[:, some]
            k, v = rows("k", "ks", i, n, some), rows("v", "vs", i, n, some)
            for h in range(hkv):
                g = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                q = s["q"][at + c:at + c + len(t), g].double()
                z = torch.einsum("tgd,jd->tgj", q, k[:, h]) * s["scale"]
                z = torch.where(keep[:, None, :], z, -math.inf)
                z = torch.softmax(z, -1)
                result["out"][at + c:at + c + len(t), g] = torch.einsum("tgj,jd->tgd", z, v[:, h])
        at += m
    return result
