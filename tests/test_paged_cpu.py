"""The C entry points of the paged operators refuse bad arguments on the host,
before a device is touched."""

import ctypes
import math
import os

import pytest

from conftest import PKG_DIR

FA_EINVAL, FA_EALIGN = 1, 2
VP, I32, I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class Cache(ctypes.Structure):
    _fields_ = [("k_pages", VP), ("v_pages", VP),
                ("k_page_stride", I64), ("k_head_stride", I64), ("k_row_stride", I64),
                ("v_page_stride", I64), ("v_head_stride", I64), ("v_row_stride", I64),
                ("page_table", VP), ("table_stride", I64), ("table_width", I32),
                ("num_pages", I32), ("page_rows", I32), ("kv_heads", I32),
                ("head_dim", I32)]


class Step(ctypes.Structure):
    _fields_ = [("starts", VP), ("seq_lens", VP), ("batch", I32), ("tokens", I32)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(PKG_DIR, "flashattn_cuda", "libfa_b200.so"))
    f, i = ctypes.c_float, ctypes.c_int
    lib.fa_rope.argtypes = [VP] * 6 + [i] * 5 + [VP, I64, VP, i, f, i, i, VP]
    lib.fa_append_paged.argtypes = ([VP] * 7 + [i, VP, VP, VP, VP, i, f, i, i, VP])
    lib.fa_attend_paged.argtypes = [VP] * 4 + [i, VP, VP, f, i, i, VP, ctypes.c_size_t,
                                               VP, ctypes.c_size_t, VP]
    lib.fa_attend_paged_workspace_bytes.restype = ctypes.c_size_t
    return lib


P = 4096


def cache(**kw):
    values = dict(k_pages=P, v_pages=P, k_page_stride=2048, k_head_stride=1024,
                  k_row_stride=64, v_page_stride=2048, v_head_stride=1024, v_row_stride=64,
                  page_table=P, table_stride=4, table_width=4, num_pages=9, page_rows=16,
                  kv_heads=2, head_dim=64)
    return Cache(**{**values, **kw})


def step(**kw):
    return Step(**{**dict(starts=P, seq_lens=P, batch=3, tokens=5), **kw})


def strides(*s):
    return (I64 * len(s))(*s)


def attend(lib, c=None, s=None, q=P, o=P, q_strides=(512, 64), h=8, scale=0.125, dtype=0,
           ws=P, counters=P):
    return lib.fa_attend_paged(q, strides(*q_strides), o, None, h,
                               ctypes.byref(c or cache()), ctypes.byref(s or step()), scale, 1,
                               dtype, ws, 1 << 30, counters, 1 << 20, None)


@pytest.mark.parametrize("kw", [
    dict(c=cache(k_pages=None)), dict(c=cache(page_table=None)), dict(c=cache(head_dim=96)),
    dict(c=cache(page_rows=12)), dict(c=cache(page_rows=0)), dict(c=cache(num_pages=0)),
    dict(c=cache(kv_heads=0)), dict(c=cache(kv_heads=3)), dict(c=cache(table_width=0)),
    dict(c=cache(table_stride=-1)), dict(c=cache(k_page_stride=0)),
    dict(c=cache(v_row_stride=-64)), dict(s=step(starts=None)), dict(s=step(batch=0)),
    dict(s=step(tokens=0)), dict(s=step(tokens=2 ** 31 - 1)), dict(q=None), dict(o=None),
    dict(ws=None), dict(counters=None), dict(h=0), dict(h=7), dict(h=2 * 129),
    dict(q_strides=(0, 64)), dict(q_strides=(512, -64)), dict(scale=math.nan),
    dict(scale=math.inf), dict(dtype=2)])
def test_attend_refuses_values(lib, kw):
    assert attend(lib, **kw) == FA_EINVAL


@pytest.mark.parametrize("kw", [
    dict(q=P + 8), dict(o=P + 2), dict(ws=P + 4), dict(q_strides=(516, 64)),
    dict(c=cache(v_pages=P + 8)), dict(c=cache(k_row_stride=68)),
    dict(c=cache(page_table=P + 2)), dict(s=step(seq_lens=P + 1)), dict(counters=P + 2)])
def test_attend_refuses_alignment(lib, kw):
    assert attend(lib, **kw) == FA_EALIGN


def rope(lib, q=P, qo=P, k=None, ko=None, b=1, h=2, hkv=1, n=4, d=64, pos=P, freqs=P, rot=64,
         amplitude=1.0, flags=0, dtype=0):
    s = strides(h * n * d, n * d, d)
    return lib.fa_rope(q, s, qo, k, s, ko, b, h, hkv, n, d, pos, 0, freqs, rot, amplitude,
                       flags, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(qo=None), 1), (dict(k=P), 1), (dict(pos=None), 1),
    (dict(freqs=None), 1), (dict(b=0), 1), (dict(h=70000), 1), (dict(n=0), 1),
    (dict(d=1026, rot=2), 1), (dict(rot=0), 1), (dict(rot=65), 1), (dict(rot=66), 1),
    (dict(b=1 << 16, n=1 << 16), 1), (dict(amplitude=math.nan), 1), (dict(flags=4), 1),
    (dict(dtype=3), 1), (dict(freqs=P + 4), 2), (dict(pos=P + 2), 2), (dict(q=P + 1), 2),
    (dict(k=P, ko=P, hkv=0), 1)])
def test_rope_refuses(lib, kw, status):
    assert rope(lib, **kw) == status


def append(lib, q=None, qo=None, k=P, v=P, h=4, c=None, s=None, freqs=None, rot=64,
           amplitude=1.0, flags=0, dtype=0):
    st = strides(512, 64)
    return lib.fa_append_paged(q, st, qo, k, st, v, st, h, ctypes.byref(c or cache()),
                               ctypes.byref(s or step()), None, freqs, rot, amplitude, flags,
                               dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), 1), (dict(v=None), 1), (dict(q=P), 1), (dict(q=P, qo=P), 1),
    (dict(q=P, qo=P, freqs=P, h=0), 1), (dict(freqs=P, rot=66), 1), (dict(freqs=P, rot=3), 1),
    (dict(flags=2), 1), (dict(dtype=7), 1), (dict(c=cache(page_rows=20)), 1),
    (dict(s=step(tokens=-1)), 1), (dict(freqs=P + 2), 2), (dict(v=P + 1), 2),
    (dict(c=cache(k_pages=P + 8)), 2)])
def test_append_refuses(lib, kw, status):
    assert append(lib, **kw) == status


def test_workspace_of_other_head_dims_is_none(lib):
    assert lib.fa_attend_paged_workspace_bytes(80, 0) == 0
