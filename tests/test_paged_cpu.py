"""Rotary positions and the paged cache without a GPU: rates, the page allocator, and what calls refuse (argument checks and
the C entries' codes come before anything is launched)."""
import ctypes
import math
import pickle

import pytest
import torch

import moda_amd
from moda_amd import _lib


def test_rates():
    f = moda_amd.Rotary(8, base=100.0).rates(torch.device("cpu"))
    assert f.dtype == torch.float64
    for i in range(4):
        assert math.isclose(float(f[i]), 100.0 ** (-i / 4) / (2 * math.pi), rel_tol=1e-14)
    lin = moda_amd.Rotary(8, base=100.0, scaling="linear", factor=4.0).rates("cpu")
    assert torch.allclose(lin * 4, f, rtol=1e-14)
    ntk = moda_amd.Rotary(8, base=100.0, scaling="ntk", factor=4.0).rates("cpu")
    assert math.isclose(float(ntk[0]), float(f[0]), rel_tol=1e-14) and math.isclose(float(ntk[3]), float(f[3]) / 4, rel_tol=1e-12)
    r = moda_amd.Rotary(64, scaling="by_parts", factor=8.0, original_length=4096)
    plain, parts = moda_amd.Rotary(64).rates("cpu"), r.rates("cpu")
    turns = plain * 4096
    assert torch.equal(parts[turns >= 32], plain[turns >= 32])
    assert torch.allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((parts < plain) & (parts > plain / 8))[between].all()
    assert math.isclose(r.amplitude, 0.1 * math.log(8.0) + 1)
    own = moda_amd.Rotary(4, rates=[0.25, 0.5], amplitude=2.0)
    assert own.rates("cpu").tolist() == [0.25, 0.5] and own.amplitude == 2.0
    again = pickle.loads(pickle.dumps(r))
    assert torch.equal(again.rates("cpu"), parts) and again.amplitude == r.amplitude


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, factor=0.0), dict(dim=8, base=-1.0),
                                dict(dim=8, scaling="by_parts", factor=2.0), dict(dim=2, scaling="ntk", factor=2.0),
                                dict(dim=8, rates=[1.0]), dict(dim=4, rates=[1.0, math.nan]),
                                dict(dim=8, scaling="by_parts", factor=2.0, original_length=10, slow=3.0, fast=3.0)], ids=str)
def test_rates_that_are_refused(kw):
    with pytest.raises(ValueError):
        moda_amd.Rotary(**kw)


def test_no_cpu_path():
    x = torch.zeros(1, 4, 2, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moda_amd.apply_rotary(x, None, moda_amd.Rotary(16))
    pages, table, past = torch.zeros(2, 16, 2, 16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moda_amd.paged_append(x, x, pages, pages, table, past)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moda_amd.paged_moda(x, pages, pages, table, past)
    with pytest.raises(RuntimeError, match="no CPU path"):
        moda_amd.paged_attn(x, pages, pages, table, past)
    with pytest.raises(ValueError):
        moda_amd.apply_rotary(None, None, moda_amd.Rotary(16))


def test_pages_are_handed_out_and_taken_back():
    c = moda_amd.PagedKVCache(2, 6, 16, 2, 8, torch.bfloat16, "cpu", batch=3, max_tokens=64)
    assert c.k.shape == (2, 6, 16, 2, 8) and c.page_table.shape == (3, 4) and (c.page_table == -1).all()
    c.reserve(0, 1)
    c.reserve(1, 33)
    c.reserve(0, 16)  # has it already
    used = [x for x in c.page_table.flatten().tolist() if x >= 0]
    assert len(used) == 4 and len(set(used)) == 4
    first = c.page_table[0].tolist()
    c.reserve(0, 17)
    assert c.page_table[0, 0] == first[0] and c.page_table[0, 1] >= 0 and c.page_table[0, 2] == -1
    c.past.copy_(torch.tensor([17, 33, 0]))
    with pytest.raises(RuntimeError, match="full"):
        c.reserve(2, 40)
    assert (c.page_table[2] == -1).all()
    with pytest.raises(ValueError):
        c.reserve(2, 65)
    c.release(1)
    assert (c.page_table[1] == -1).all() and c.past.tolist() == [17, 0, 0]
    c.reserve(2, 64)
    used = [x for x in c.page_table.flatten().tolist() if x >= 0]
    assert len(used) == 6 and len(set(used)) == 6
    c.advance(torch.tensor([1, 0, 5], dtype=torch.int32))
    assert c.past.tolist() == [18, 0, 5]
    c.advance(1)
    assert c.past.tolist() == [19, 1, 6]
    for bad in (dict(page_size=24), dict(page_size=0), dict(n_pages=0), dict(batch=0), dict(max_tokens=0), dict(layers=0)):
        kw = dict(layers=1, n_pages=2, page_size=16, H=1, D=8, dtype=torch.float32, device="cpu")
        kw.update(bad)
        with pytest.raises(ValueError):
            moda_amd.PagedKVCache(**kw)


class Rot(ctypes.Structure):
    _fields_ = [("rates", ctypes.c_void_p), ("dim", ctypes.c_int64), ("amplitude", ctypes.c_float), ("interleaved", ctypes.c_int32),
                ("inverse", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class Part(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("y", ctypes.c_void_p), ("sx", _lib.Strides), ("sy", _lib.Strides), ("rows", ctypes.c_int64),
                ("heads", ctypes.c_int64)]


class PagesC(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("dtype", ctypes.c_int32)] + \
        [(n, ctypes.c_int64) for n in ("B", "T", "H", "D", "Dv", "n_pages", "page_size", "max_pages")] + \
        [("k_pages", ctypes.c_void_p), ("v_pages", ctypes.c_void_p), ("k", _lib.Strides), ("v", _lib.Strides), ("table", ctypes.c_void_p),
         ("table_stride", ctypes.c_int64), ("past", ctypes.c_void_p), ("new_lens", ctypes.c_void_p), ("cu_seqlens", ctypes.c_void_p),
         ("total_tokens", ctypes.c_int64)]


class AppendC(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("reserved", ctypes.c_int32)] + \
        [(n, ctypes.c_void_p) for n in ("k", "v", "q", "q_out", "kd", "vd")] + \
        [(n, _lib.Strides) for n in ("sk", "sv", "sq", "sq_out", "skd", "svd")] + [(n, ctypes.c_int64) for n in ("G", "Hq", "L", "slot")]


class AttendC(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_int32), ("plain", ctypes.c_int32)] + [(n, ctypes.c_void_p) for n in ("q", "kd", "vd", "o", "lse")] + \
        [(n, _lib.Strides) for n in ("sq", "skd", "svd", "so")] + [(n, ctypes.c_int64) for n in ("G", "L", "L_valid")] + \
        [("scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = -1, -2, -3, -4
AT = 1 << 20  # an address that nothing is read from: every call below is refused before it, or has nothing to do


def strides(*x):
    return _lib.Strides(*x)


def pages(**kw):
    c = PagesC(struct_size=ctypes.sizeof(PagesC), dtype=_lib.BF16, B=2, T=1, H=2, D=64, Dv=64, n_pages=4, page_size=16, max_pages=3,
               k_pages=AT, v_pages=AT, k=strides(2048, 128, 64), v=strides(2048, 128, 64), table=AT, table_stride=3, past=AT)
    for n, x in kw.items():
        setattr(c, n, x)
    return c


def test_c_entries_refuse_rotations():
    lib = _lib.load()
    s = strides(64, 64, 64)

    def call(dtype=_lib.BF16, B=1, T=1, D=64, n=1, part=None, rot=None, pos=None, pos64=0, ps=0):
        p = Part(AT, AT, s, s, 1, 1)
        for k, v in (part or {}).items():
            setattr(p, k, v)
        r = Rot(AT, 64, 1.0, 0, 0, 0)
        for k, v in (rot or {}).items():
            setattr(r, k, v)
        i64 = ctypes.c_int64
        return lib.moda_hip_rotary_rows(dtype, i64(B), i64(T), i64(D), ctypes.byref(p), n, ctypes.c_void_p(pos), pos64, i64(ps), ctypes.byref(r), None)

    assert call(B=0) == 0
    for kw in (dict(dtype=3), dict(B=-1), dict(T=-1), dict(D=0), dict(n=0), dict(n=4), dict(ps=-1), dict(rot=dict(rates=None)), dict(rot=dict(dim=0)),
               dict(rot=dict(dim=7)), dict(rot=dict(dim=66)), dict(part=dict(x=None)), dict(part=dict(y=None)), dict(part=dict(rows=0)),
               dict(part=dict(heads=0))):
        assert call(**kw) == EINVAL, kw
    for kw in (dict(T=1 << 31), dict(B=1 << 20, T=1 << 20), dict(D=516, rot=dict(dim=64)), dict(part=dict(rows=1 << 15)), dict(part=dict(heads=1 << 20))):
        assert call(**kw) == EUNSUPPORTED, kw
    for kw in (dict(part=dict(x=AT + 1)), dict(part=dict(y=AT + 1)), dict(rot=dict(rates=AT + 4)), dict(pos=AT + 2), dict(pos=AT + 4, pos64=1)):
        assert call(**kw) == EALIGN, kw


BAD_PAGES = [
    (EINVAL, dict(struct_size=8)), (EINVAL, dict(dtype=7)), (EINVAL, dict(B=-1)), (EINVAL, dict(T=-1)), (EINVAL, dict(H=0)), (EINVAL, dict(D=0)),
    (EINVAL, dict(Dv=0)), (EINVAL, dict(n_pages=0)), (EINVAL, dict(max_pages=0)), (EINVAL, dict(page_size=0)), (EINVAL, dict(table_stride=-1)),
    (EINVAL, dict(k_pages=None)), (EINVAL, dict(v_pages=None)), (EINVAL, dict(table=None)), (EINVAL, dict(past=None)),
    (EINVAL, dict(new_lens=AT, cu_seqlens=AT)),
    (EUNSUPPORTED, dict(D=264)), (EUNSUPPORTED, dict(Dv=264)), (EUNSUPPORTED, dict(D=12)), (EUNSUPPORTED, dict(Dv=60)),
    (EUNSUPPORTED, dict(page_size=24)), (EUNSUPPORTED, dict(n_pages=1 << 27)), (EUNSUPPORTED, dict(max_pages=1 << 27)), (EUNSUPPORTED, dict(max_pages=(1 << 26) + 1)), (EUNSUPPORTED, dict(page_size=1, max_pages=1 << 28)),
    (EUNSUPPORTED, dict(n_pages=1 << 62)), (EUNSUPPORTED, dict(T=1 << 24)), (EUNSUPPORTED, dict(B=1 << 20)),
    (EALIGN, dict(k_pages=AT + 8)), (EALIGN, dict(v_pages=AT + 2)), (EALIGN, dict(k=strides(2048, 128, 60))), (EALIGN, dict(v=strides(2049, 128, 64))),
    (EALIGN, dict(table=AT + 1)), (EALIGN, dict(past=AT + 2)), (EALIGN, dict(new_lens=AT + 3)),
]


@pytest.mark.parametrize("code,kw", BAD_PAGES, ids=str)
def test_c_entries_refuse_caches(code, kw):
    lib = _lib.load()
    lib.moda_hip_paged_attend_workspace_bytes.restype = ctypes.c_size_t
    s = strides(128, 128, 64)
    a = AppendC(struct_size=ctypes.sizeof(AppendC), k=AT, v=AT, sk=s, sv=s)
    t = AttendC(struct_size=ctypes.sizeof(AttendC), q=AT, o=AT, lse=AT, sq=s, so=s, G=1, scale=1.0)
    c = pages(**kw)
    assert lib.moda_hip_paged_append(ctypes.byref(c), ctypes.byref(a), None, None) == code
    assert lib.moda_hip_paged_attend_workspace_bytes(ctypes.byref(c), ctypes.byref(t)) == 0
    assert lib.moda_hip_paged_attend(ctypes.byref(c), ctypes.byref(t), AT, ctypes.c_size_t(1 << 40), None) == code


def test_c_entries_refuse_appends_and_attentions():
    lib = _lib.load()
    s = strides(128, 128, 64)

    def append(c=None, rot=None, **kw):
        a = AppendC(struct_size=ctypes.sizeof(AppendC), k=AT, v=AT, sk=s, sv=s, sq=s, sq_out=s, skd=s, svd=s, G=1, Hq=2, L=4, slot=0)
        for n, x in kw.items():
            setattr(a, n, x)
        return lib.moda_hip_paged_append(ctypes.byref(pages(**(c or {}))), ctypes.byref(a), ctypes.byref(rot) if rot else None, None)

    assert append(c=dict(B=0)) == 0 and append(c=dict(T=0)) == 0 and append(c=dict(cu_seqlens=AT, total_tokens=0)) == 0
    for kw in (dict(struct_size=4), dict(kd=AT), dict(kd=AT, vd=AT, L=0), dict(kd=AT, vd=AT, slot=4), dict(kd=AT, vd=AT, slot=-1), dict(q=AT, G=0, q_out=AT),
               dict(q=AT, Hq=0, q_out=AT), dict(q=AT), dict(k=None), dict(v=None), dict(rot=Rot(AT, 66, 1.0, 0, 0, 0)), dict(rot=Rot(None, 64, 1.0, 0, 0, 0))):
        assert append(**kw) == EINVAL, kw
    assert append(q=AT, q_out=AT, G=1 << 15) == EUNSUPPORTED and append(kd=AT, vd=AT, L=1 << 20) == EUNSUPPORTED
    assert append(k=AT + 1) == EALIGN and append(q=AT, q_out=AT + 1) == EALIGN

    def attend(c=None, ws=AT, **kw):
        t = AttendC(struct_size=ctypes.sizeof(AttendC), q=AT, o=AT, lse=AT, sq=s, so=s, skd=s, svd=s, G=1, scale=1.0)
        for n, x in kw.items():
            setattr(t, n, x)
        return lib.moda_hip_paged_attend(ctypes.byref(pages(**(c or {}))), ctypes.byref(t), ws, ctypes.c_size_t(1 << 40 if ws else 0), None)

    assert attend(c=dict(B=0)) == 0 and attend(c=dict(T=0)) == 0
    for kw in (dict(struct_size=4), dict(G=0), dict(L=-1), dict(L=2, L_valid=3, kd=AT, vd=AT), dict(L=2), dict(L=2, kd=AT), dict(plain=1, L=2, kd=AT, vd=AT),
               dict(q=None), dict(o=None), dict(lse=None), dict(c=dict(cu_seqlens=AT))):
        assert attend(**kw) == EINVAL, kw
    for kw in (dict(G=1 << 15), dict(c=dict(T=1 << 20), G=1 << 10), dict(L=1 << 20, kd=AT, vd=AT)):
        assert attend(**kw) == EUNSUPPORTED, kw
    for kw in (dict(q=AT + 2), dict(o=AT + 8), dict(lse=AT + 2), dict(L=2, kd=AT + 2, vd=AT), dict(sq=strides(128, 128, 63)), dict(ws=AT + 4)):
        assert attend(**kw) == EALIGN, kw
    assert attend(ws=None) == EWORKSPACE
