"""What the 8-bit cache and windowed attention refuse: on the host, before any launch."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    from vllm_apple_b200 import _lib
    return _lib.load()


def _decode(lib, **kw):
    a = dict(out=16, q=16, kc=16, vc=16, ks=16, vs=16, e4m3=1, bt=16, sl=16, nk=None, nv=None, B=4,
             Hq=32, Hkv=8, D=128, bs=16, mb=8, max_len=128, nb=64, scale=0.1, window=0, sinks=0,
             sb=16384, sh=2048, st=128, cb=128, ch=16, ct=1, qt=4096, qh=128, ot=4096, oh=128,
             nt=1024, nh=128, ws=None, wsb=0)
    a.update(kw)
    ptr = lambda n: None if a[n] is None else P(a[n])  # noqa: E731
    return lib.va_window_decode(
        *map(ptr, ("out", "q", "kc", "vc", "ks", "vs")), a["e4m3"],
        *map(ptr, ("bt", "sl", "nk", "nv")),
        *[a[n] for n in ("B", "Hq", "Hkv", "D", "bs", "mb", "max_len", "nb", "scale", "window",
                         "sinks", "sb", "sh", "st", "cb", "ch", "ct", "qt", "qh", "ot", "oh",
                         "nt", "nh")], ptr("ws"), a["wsb"], None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(Hkv=5), 1), (dict(Hkv=0), 1), (dict(B=-1), 1), (dict(max_len=-1), 1), (dict(sinks=-1), 1),
    (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(bs=0), 1), (dict(q=None), 1), (dict(ks=None), 1),
    (dict(nk=16), 1), (dict(q=8), 1), (dict(out=17), 1), (dict(st=120), 1), (dict(qh=100), 1),
    (dict(e4m3=0, st=132), 1), (dict(nk=16, nv=8), 1), (dict(nk=16, nv=16, nt=1004), 1),
    (dict(D=80), 2), (dict(D=256), 2), (dict(B=65536), 2), (dict(max_len=1 << 31), 2),
    (dict(B=1, max_len=100000), 4), (dict(B=0), 0), (dict(max_len=0), 0)])
def test_window_decode_refuses(lib, kw, status):
    assert _decode(lib, **kw) == status


def test_window_decode_workspace(lib):
    f = lib.va_window_decode_workspace_size
    assert f(0, 32, 8, 128, 4096, 0, 0) == 0
    assert f(4, 32, 5, 128, 4096, 0, 0) == 0
    assert f(4096, 32, 8, 128, 8192, 0, 0) == 0      # enough sequences: none is cut
    assert f(1, 32, 8, 128, 64, 0, 0) == 0           # too short to cut
    big = f(1, 32, 8, 128, 131072, 0, 0)
    assert big > 0 and big % 256 == 0
    # a short window bounds what there is to cut, however long the sequences
    assert f(1, 32, 8, 128, 1 << 30, 64, 4) == 0
    assert 0 < f(1, 32, 8, 128, 1 << 30, 1000, 4) < big


def _write(lib, D=128, T=4, H=8, bs=16, nb=64, ptr=16, st=(16384, 2048, 128), new=(1024, 128)):
    return lib.va_kv_quant_write_slots(*[P(ptr) if ptr else None] * 7, 1, T, H, D, bs, nb, *st, 128,
                                       16, 1, *new, None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), 1), (dict(H=0), 1), (dict(bs=0), 1), (dict(nb=-1), 1), (dict(ptr=None), 1),
    (dict(ptr=24), 1), (dict(st=(16384, 2048, 136)), 1), (dict(new=(1024, 100)), 1),
    (dict(D=48), 2), (dict(T=0, ptr=None), 0)])
def test_quant_write_refuses(lib, kw, status):
    assert _write(lib, **kw) == status


def _read(lib, D=128, S=4, mb=8, H=8, bs=16, ptr=16, st=(16384, 2048, 128),
          dst=(16384, 2048, 128)):
    p = P(ptr) if ptr else None
    return lib.va_kv_dequant_blocks(p, p, p, p, p, p, p, None, p, S, mb, H, D, bs, 64, 64, *st, 128,
                                    16, 1, *dst, None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(S=-1), 1), (dict(mb=-1), 1), (dict(H=0), 1), (dict(bs=0), 1), (dict(ptr=None), 1),
    (dict(ptr=8), 1), (dict(st=(16384, 2048, 72)), 1), (dict(dst=(16384, 2048, 100)), 1),
    (dict(D=80), 2), (dict(bs=1 << 24), 2), (dict(S=0, ptr=None), 0), (dict(mb=0, ptr=None), 0)])
def test_dequant_refuses(lib, kw, status):
    assert _read(lib, **kw) == status


# ---- the Python layer: checks that need no device -----------------------------
def test_ops_refuse_cpu_tensors():
    from vllm_apple_b200 import ops
    k = torch.zeros(2, 2, 16, 64).to(torch.float8_e4m3fn)
    e = torch.zeros(2, 2, 16, dtype=torch.uint8)
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv_quant_write_slots(k, k, e, e, x, x, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_window_decode(x, x, k, k, None, None, scale=1.0, max_seq_len=1)


def test_cache_checks():
    from vllm_apple_b200.ops import _window_cache
    f8, f16 = torch.float8_e4m3fn, torch.float16
    k8, e = torch.zeros(3, 2, 16, 64).to(f8), torch.zeros(3, 2, 16, dtype=torch.uint8)
    k16 = torch.zeros(3, 2, 16, 64, dtype=f16)
    q8, g, sc = _window_cache(k8, k8, e, e, "hnd")
    # (blocks, heads, block size, head size, strides of block, head and token)
    assert q8 and g == (3, 2, 16, 64, 2048, 1024, 64) and sc == (32, 16, 1)
    q8, g, sc = _window_cache(k8, k8, e, e, "nhd")
    assert g == (3, 16, 2, 64, 2048, 64, 1024) and sc == (32, 1, 16)
    assert not _window_cache(k16, k16, None, None, "hnd")[0]
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        _window_cache(k16.float(), k16.float(), None, None, "hnd")
    with pytest.raises(ValueError, match="layout"):
        _window_cache(k16, k16, None, None, "dhn")
    with pytest.raises(ValueError, match="4-D"):
        _window_cache(k16[0], k16[0], None, None, "hnd")
    with pytest.raises(ValueError, match="contiguous"):
        _window_cache(k16.transpose(2, 3), k16.transpose(2, 3), None, None, "hnd")
    with pytest.raises(ValueError, match="differ"):
        _window_cache(k16, k16[:2], None, None, "hnd")
    with pytest.raises(ValueError, match="differ"):
        _window_cache(k8, k16, e, e, "hnd")
    with pytest.raises(ValueError, match="belong"):
        _window_cache(k16, k16, e, e, "hnd")
    with pytest.raises(ValueError, match="needs"):
        _window_cache(k8, k8, e, None, "hnd")
    with pytest.raises(TypeError, match="uint8"):
        _window_cache(k8, k8, e.int(), e, "hnd")
    with pytest.raises(ValueError, match="first three"):
        _window_cache(k8, k8, e[:, :1], e, "hnd")
    with pytest.raises(ValueError, match="strides"):
        _window_cache(k8, k8, e, e.transpose(0, 0).clone().as_strided(e.shape, (32, 1, 2)), "hnd")


def test_new_row_and_table_checks():
    from vllm_apple_b200.ops import _ints, _new_rows, _table
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    assert _new_rows(x, x, 2, 64, 3) == (128, 64)
    for bad in (x[:2], x[:, :1], x[..., :32], x.transpose(1, 2)):
        with pytest.raises(ValueError):
            _new_rows(bad, bad, 2, 64, 3)
    with pytest.raises(ValueError):
        _new_rows(x, None, 2, 64, 3)
    with pytest.raises(ValueError):
        _new_rows(x, torch.zeros(3, 4, 64, dtype=torch.float16)[:, ::2], 2, 64, 3)
    with pytest.raises(TypeError):
        _new_rows(x.float(), x.float(), 2, 64, 3)
    v = torch.zeros(6, dtype=torch.int32)
    _ints(v, "v", 6)
    for bad in (v[:5], v[::2]):
        with pytest.raises(ValueError):
            _ints(bad, "v", 6)
    with pytest.raises(TypeError):
        _ints(v.long(), "v", 6)
    t = torch.zeros(2, 5, dtype=torch.int32)
    assert _table(t, 2) == 5
    for bad in (t[:1], t[0], torch.zeros(5, 2, dtype=torch.int32).t()):
        with pytest.raises(ValueError):
            _table(bad, 2)
    with pytest.raises(TypeError):
        _table(t.long(), 2)
