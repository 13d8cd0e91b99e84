"""Rotary positions and attention's training pair refuse invalid arguments with the documented codes,
before anything touches a GPU (no pointer here is ever dereferenced on the device)."""
import ctypes
import math

import pytest

import tsa

P = 0x10000  # an aligned address that nothing reads


def rows(data=P, b=1 << 16, h=1 << 12, t=64):
    return tsa.TsaRows(data, b, h, t)


def ref(x):
    return None if x is None else ctypes.byref(x)


def params(**kw):
    f = dict(base=1e4, factor=1.0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0, rot=64, scaling=0, orig_len=0)
    f.update(kw)
    return tsa.TsaRopeParams(**f)


def freqs(p, table=None, amp=None):
    table = (ctypes.c_uint64 * max(1, p.rot // 2))() if table is None else table
    amp = ctypes.c_float() if amp is None else amp
    return tsa.load().tsa_rope_freqs(ctypes.addressof(p), ctypes.addressof(table), ctypes.addressof(amp))


def test_freqs_refusals():
    lib, good = tsa.load(), params()
    assert freqs(good) == tsa.TSA_OK
    assert lib.tsa_rope_freqs(None, P, P) == tsa.TSA_ERR_NULL
    assert lib.tsa_rope_freqs(ctypes.addressof(good), None, P) == tsa.TSA_ERR_NULL
    assert lib.tsa_rope_freqs(ctypes.addressof(good), P, None) == tsa.TSA_ERR_NULL
    for rot in (0, -2, 1, 63):
        assert freqs(params(rot=rot)) == tsa.TSA_ERR_SHAPE
    for bad in (dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(scaling=5), dict(scaling=-1), dict(scaling=1, factor=0.5),
                dict(scaling=1, factor=math.nan), dict(scaling=1, factor=math.inf), dict(scaling=2, factor=2.0, rot=2),
                dict(scaling=3, factor=2.0), dict(scaling=4, factor=2.0), dict(scaling=3, factor=2.0, orig_len=10, beta_fast=1.0),
                dict(scaling=3, factor=2.0, orig_len=10, beta_slow=0.0), dict(scaling=3, factor=2.0, orig_len=10, beta_fast=math.inf),
                dict(scaling=4, factor=2.0, orig_len=10, high=1.0), dict(scaling=4, factor=2.0, orig_len=10, low=0.0)):
        assert freqs(params(**bad)) == tsa.TSA_ERR_ARG, bad


def test_freqs_table():
    """The first pair turns a radian a position: 2^64 / 2 pi; the others fall by base^(-2 / rot)."""
    table, amp = (ctypes.c_uint64 * 32)(), ctypes.c_float(-1)
    assert freqs(params(), table, amp) == tsa.TSA_OK and amp.value == 1.0
    assert abs(table[0] - 2935890503282001226) <= 1  # 2^64 / (2 pi) = 2935890503282001226.4...
    for i in range(32):
        assert table[i] == pytest.approx(2 ** 64 / (2 * math.pi) * 1e4 ** (-i / 32), rel=1e-14)
    assert freqs(params(scaling=3, factor=16.0, orig_len=4096), table, amp) == tsa.TSA_OK
    assert amp.value == pytest.approx(0.1 * math.log(16) + 1, rel=2.0 ** -23)


def plan(**kw):
    f = dict(freq=P, amp=1.0, rot=64, interleaved=0)
    f.update(kw)
    return tsa.TsaRopePlan(**f)


def rope(p=plan(), type=tsa.TSA_TYPE_F16, q=rows(), qo=rows(2 * P), Hq=4, k=rows(), ko=rows(2 * P), Hk=2, B=2, T=3, D=64, back=0):
    return tsa.load().tsa_rope(ref(p), type, ref(q), ref(qo), Hq, ref(k), ref(ko), Hk, None, None, None, B, T, D, back, None)


def test_rope_refusals():
    assert rope(p=None) == tsa.TSA_ERR_NULL and rope(p=plan(freq=None)) == tsa.TSA_ERR_NULL
    for kw in (dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(q=rows(None)), dict(ko=rows(None))):
        assert rope(**kw) == tsa.TSA_ERR_NULL, kw
    for kw in (dict(B=0), dict(T=0), dict(Hq=0), dict(Hk=-1), dict(D=0), dict(p=plan(rot=0)), dict(p=plan(rot=65)), dict(p=plan(rot=66)),
               dict(p=plan(rot=7)), dict(B=1 << 20, T=1 << 10), dict(Hq=65535)):
        assert rope(**kw) == tsa.TSA_ERR_SHAPE, kw
    for D in (32, 96, 512):
        assert rope(D=D) == tsa.TSA_ERR_UNSUPPORTED
    for kw in (dict(p=plan(interleaved=2)), dict(p=plan(amp=math.nan)), dict(p=plan(amp=math.inf)), dict(type=2), dict(back=2), dict(q=rows(P + 8)),
               dict(q=rows(t=63)), dict(qo=rows(2 * P, t=0)), dict(k=rows(h=-8)), dict(q=rows(P), qo=rows(P, t=128)), dict(ko=rows(P, b=8))):
        assert rope(**kw) == tsa.TSA_ERR_ARG, kw


def fwd(q=rows(), k=rows(), v=rows(), gate=None, o=rows(), lse=P, B=2, Hq=4, Hkv=2, Tq=3, Tk=5, D=64, scale=0.1, causal=1):
    return tsa.load().tsa_attn_train_fwd(ref(q), ref(k), ref(v), ref(gate), ref(o), lse, None, None, B, Hq, Hkv, Tq, Tk, D, scale, causal, None)


def bwd(do=rows(), q=rows(), k=rows(), v=rows(), gate=None, o=rows(), lse=P, dq=rows(), dk=rows(), dv=rows(), dgate=None, B=2, Hq=4,
        Hkv=2, Tq=3, Tk=5, D=64, scale=0.1, causal=1, ws=P, n=1 << 40):
    return tsa.load().tsa_attn_bwd(ref(do), ref(q), ref(k), ref(v), ref(gate), ref(o), lse, ref(dq), ref(dk), ref(dv), ref(dgate), None, None,
                                   B, Hq, Hkv, Tq, Tk, D, scale, causal, ws, n, None)


@pytest.mark.parametrize("call", [fwd, bwd], ids=lambda f: f.__name__)
def test_pair_refusals(call):
    names = ["q", "k", "v", "o"] + (["do", "dq", "dk", "dv"] if call is bwd else [])
    for name in names:
        assert call(**{name: None}) == tsa.TSA_ERR_NULL, name
        assert call(**{name: rows(None)}) == tsa.TSA_ERR_NULL, name
        assert call(**{name: rows(P + 8)}) == tsa.TSA_ERR_ARG, name
        assert call(**{name: rows(t=60)}) == tsa.TSA_ERR_ARG, name
        assert call(**{name: rows(h=-8)}) == tsa.TSA_ERR_ARG, name
        assert call(**{name: rows(t=(1 << 24) + 8)}) == tsa.TSA_ERR_SHAPE, name
    for name in ["o"] if call is fwd else ["dq", "dk", "dv"]:
        assert call(**{name: rows(t=0)}) == tsa.TSA_ERR_ARG, name
    assert call(lse=None) == tsa.TSA_ERR_NULL
    assert call(gate=rows(P + 2), **({"dgate": rows()} if call is bwd else {})) == tsa.TSA_ERR_ARG
    for name in ("B", "Hq", "Hkv", "Tq", "Tk", "D"):
        assert call(**{name: 0}) == tsa.TSA_ERR_SHAPE, name
        assert call(**{name: -1}) == tsa.TSA_ERR_SHAPE, name
    assert call(Hq=3) == tsa.TSA_ERR_SHAPE
    assert call(Tq=1 << 30) == tsa.TSA_ERR_SHAPE
    assert call(Tk=1 << 30) == tsa.TSA_ERR_SHAPE
    assert call(B=1, Hq=1, Hkv=1, Tq=1 << 30, Tk=(1 << 30) + 1) == tsa.TSA_ERR_SHAPE
    for D in (32, 96, 192, 512):
        assert call(D=D) == tsa.TSA_ERR_UNSUPPORTED
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert call(scale=scale) == tsa.TSA_ERR_ARG
    for causal in (2, -1):
        assert call(causal=causal) == tsa.TSA_ERR_ARG


def test_backward_workspace():
    lib = tsa.load()
    need = lib.tsa_attn_bwd_workspace_bytes(2, 4, 2, 3, 5, 64, 0, 1)
    assert need > 0
    assert bwd(ws=None) == tsa.TSA_ERR_WORKSPACE
    assert bwd(n=need - 1) == tsa.TSA_ERR_WORKSPACE
    assert bwd(ws=P + 8) == tsa.TSA_ERR_ARG
    assert bwd(gate=rows()) == tsa.TSA_ERR_NULL  # no dgate
    more = lib.tsa_attn_bwd_workspace_bytes(2, 4, 2, 3, 5, 64, 1, 1)
    assert more >= need + 2 * 4 * 3 * 64 * 2
    assert bwd(gate=rows(), dgate=rows(), n=more - 1) == tsa.TSA_ERR_WORKSPACE
    for bad in ((0, 4, 2, 3, 5, 64, 0, 1), (2, 3, 2, 3, 5, 64, 0, 1), (2, 4, 2, 3, 5, 96, 0, 1), (2, 4, 2, 3, 5, 64, 2, 1), (2, 4, 2, 3, 5, 64, 0, 2),
                (2, 4, 2, 1 << 30, 5, 64, 0, 1)):
        assert lib.tsa_attn_bwd_workspace_bytes(*bad) == 0, bad


@pytest.mark.parametrize("call", [fwd, bwd], ids=lambda f: f.__name__)
def test_pair_of_too_many_rows(call):
    """More blocks of 32 rows than a launch has threads for."""
    assert call(B=1 << 22, Hq=1, Hkv=1, Tq=1, Tk=1) == tsa.TSA_ERR_SHAPE
    assert call(B=1, Hq=1, Hkv=1, Tq=1 << 27, Tk=1 << 27) == tsa.TSA_ERR_SHAPE
    assert tsa.load().tsa_attn_bwd_workspace_bytes(1 << 22, 1, 1, 1, 1, 64, 0, 1) == 0
    assert tsa.load().tsa_attn_bwd_workspace_bytes((1 << 22) - 1, 1, 1, 1, 1, 64, 0, 1) > 0
