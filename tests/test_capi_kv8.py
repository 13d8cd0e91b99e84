"""The 8-bit K/V cache's entry points refuse invalid arguments with the documented codes, before
anything touches a GPU (no pointer here is ever dereferenced on the device)."""
import ctypes

import pytest

import tsa

P = 0x10000  # an aligned address that nothing reads


def cache(**kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, k_sum=P, k_sum_scale=P, k_open=P, v_open=P, table=P, B=2, Hkv=2, D=64, n_pages=8,
             max_blocks=4)
    f.update(kw)
    return tsa.TsaKv8(**f)


def rows(data=P, b=1024, h=512, t=64):
    return tsa.TsaRows(data, b, h, t)


def ref(x):
    return None if x is None else ctypes.byref(x)


def write(c=None, k=None, v=None, n=P, T=3):
    return tsa.load().tsa_kv8_write(ref(c or cache()), ref(k or rows()), ref(v or rows()), n, None, T, None)


def read(c=None, k=rows(), v=rows(), n=P, S=3):
    return tsa.load().tsa_kv8_read(ref(c or cache()), n, None, S, ref(k), ref(v), None)


def attn(c=None, q=None, o=None, gate=None, n=P, T=3, Hq=4, max_len=256, scale=0.1, causal=1, ws=P, ws_bytes=1 << 40):
    return tsa.load().tsa_attn_kv8_fwd(ref(c or cache()), ref(q or rows()), ref(gate), ref(o or rows()), n, None, T, Hq, max_len,
                                       scale, causal, ws, ws_bytes, None)


def select(c=None, q=None, n=P, T=3, Hq=4, top=4, first=1, recent=1, blocks=P, max_len=256, ws=P, ws_bytes=1 << 40):
    return tsa.load().tsa_kv8_select(ref(c or cache()), ref(q or rows()), n, None, T, Hq, top, first, recent, blocks, max_len, ws,
                                     ws_bytes, None)


def sparse(c=None, q=None, o=None, n=P, T=3, Hq=4, blocks=P, top=4, scale=0.1, ws=P, ws_bytes=1 << 40):
    return tsa.load().tsa_attn_kv8_blocks_fwd(ref(c or cache()), ref(q or rows()), None, ref(o or rows()), n, None, T, Hq, blocks, top,
                                              scale, ws, ws_bytes, None)


CALLS = [write, read, attn, select, sparse]


@pytest.mark.parametrize("call", CALLS, ids=lambda f: f.__name__)
def test_cache_fields(call):
    for name in ("k", "v", "k_scale", "v_scale", "k_sum", "k_sum_scale", "k_open", "v_open", "table"):
        assert call(cache(**{name: None})) == tsa.TSA_ERR_NULL, name
    for name in ("B", "Hkv", "D", "n_pages", "max_blocks"):
        assert call(cache(**{name: 0})) == tsa.TSA_ERR_SHAPE, name
        assert call(cache(**{name: -1})) == tsa.TSA_ERR_SHAPE, name
    for D in (32, 96, 192, 512):
        assert call(cache(D=D)) == tsa.TSA_ERR_UNSUPPORTED
    for name in ("k", "v", "k_sum", "k_open", "v_open"):
        assert call(cache(**{name: P + 8})) == tsa.TSA_ERR_ARG, name
    assert call(cache(max_blocks=1 << 26)) == tsa.TSA_ERR_SHAPE
    assert call(cache(B=65536)) == tsa.TSA_ERR_SHAPE
    assert call(cache(B=1 << 20, Hkv=1 << 20)) == tsa.TSA_ERR_SHAPE
    assert call(n=None) == tsa.TSA_ERR_NULL


def test_rows_fields():
    lib = tsa.load()
    assert lib.tsa_kv8_write(ref(cache()), None, ref(rows()), P, None, 3, None) == tsa.TSA_ERR_NULL
    assert lib.tsa_kv8_write(None, ref(rows()), ref(rows()), P, None, 3, None) == tsa.TSA_ERR_NULL
    for bad in (rows(P + 2), rows(t=63), rows(h=4), rows(b=-8)):
        assert write(k=bad) == tsa.TSA_ERR_ARG
        assert write(v=bad) == tsa.TSA_ERR_ARG
        assert attn(q=bad) == tsa.TSA_ERR_ARG
        assert attn(gate=bad) == tsa.TSA_ERR_ARG
        assert attn(o=bad) == tsa.TSA_ERR_ARG
        assert select(q=bad) == tsa.TSA_ERR_ARG
        assert sparse(q=bad) == tsa.TSA_ERR_ARG
        assert read(k=bad) == tsa.TSA_ERR_ARG
    assert write(k=rows(None)) == tsa.TSA_ERR_NULL
    # rows of an output that lie on each other
    assert attn(o=rows(h=0)) == tsa.TSA_ERR_ARG
    assert read(v=rows(t=0)) == tsa.TSA_ERR_ARG
    assert read(None, None, None) == tsa.TSA_ERR_NULL


def test_sizes():
    assert write(T=0) == tsa.TSA_ERR_SHAPE
    assert read(S=0) == tsa.TSA_ERR_SHAPE
    assert write(T=(1 << 31) - 1) == tsa.TSA_ERR_SHAPE
    for call in (attn, select, sparse):
        assert call(T=0) == tsa.TSA_ERR_SHAPE
        assert call(Hq=0) == tsa.TSA_ERR_SHAPE
        assert call(Hq=3) == tsa.TSA_ERR_SHAPE  # no multiple of the K/V heads
        assert call(T=1 << 30) == tsa.TSA_ERR_SHAPE
        assert call(cache(B=1, Hkv=1), T=1, Hq=65537) == tsa.TSA_ERR_SHAPE
    assert attn(max_len=0) == tsa.TSA_ERR_SHAPE
    assert select(max_len=0) == tsa.TSA_ERR_SHAPE
    assert select(top=0) == tsa.TSA_ERR_SHAPE
    assert sparse(top=0) == tsa.TSA_ERR_SHAPE
    assert select(top=(1 << 24) + 1) == tsa.TSA_ERR_SHAPE
    assert sparse(top=(1 << 31) - 1) == tsa.TSA_ERR_SHAPE
    assert select(first=-1) == tsa.TSA_ERR_SHAPE


def test_values():
    assert attn(causal=2) == tsa.TSA_ERR_ARG
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attn(scale=scale) == tsa.TSA_ERR_ARG
        assert sparse(scale=scale) == tsa.TSA_ERR_ARG
    assert select(top=3, first=1, recent=2) == tsa.TSA_ERR_ARG
    assert select(blocks=None) == tsa.TSA_ERR_NULL
    assert sparse(blocks=None) == tsa.TSA_ERR_NULL


def test_workspace():
    c = cache(B=1, Hkv=1, max_blocks=1 << 14, n_pages=1 << 14)
    lib = tsa.load()
    need = lib.tsa_kv8_workspace_bytes(ref(c), 1, 8, 1 << 20, 0)
    assert need > 0
    assert attn(c, T=1, Hq=8, max_len=1 << 20, ws_bytes=need - 1) == tsa.TSA_ERR_WORKSPACE
    assert attn(c, T=1, Hq=8, max_len=1 << 20, ws=None) == tsa.TSA_ERR_WORKSPACE
    top = lib.tsa_kv8_workspace_bytes(ref(c), 1, 8, 1 << 20, 64)
    assert top >= 4 << 14  # a score for each block
    assert select(c, T=1, Hq=8, max_len=1 << 20, top=64, ws_bytes=top - 1) == tsa.TSA_ERR_WORKSPACE
    assert sparse(c, T=1, Hq=8, top=64, ws=None) == tsa.TSA_ERR_WORKSPACE
    assert attn(c, T=1, Hq=8, max_len=1 << 20, ws=P + 8, ws_bytes=need) == tsa.TSA_ERR_ARG
    assert select(c, T=1, Hq=8, max_len=1 << 20, top=64, ws=P + 4, ws_bytes=top) == tsa.TSA_ERR_ARG
    assert sparse(c, T=1, Hq=8, top=64, ws=P + 8) == tsa.TSA_ERR_ARG
    for bad in (dict(T=0), dict(Hq=0), dict(max_len=0), dict(top=-1)):
        a = dict(T=1, Hq=8, max_len=64, top=0)
        a.update(bad)
        assert lib.tsa_kv8_workspace_bytes(ref(c), a["T"], a["Hq"], a["max_len"], a["top"]) == 0


def test_workspace_serves_shorter_lengths():
    """A workspace sized for the longest sequences serves calls with a smaller max_len."""
    lib = tsa.load()
    for D in (64, 128, 256):
        for B, Hkv, Hq, T in ((1, 4, 24, 1), (3, 2, 8, 2), (32, 4, 24, 1), (7, 1, 1, 1), (100, 3, 9, 1), (42, 1, 1, 200), (6, 7, 7, 200), (2, 5, 20, 33)):
            c = cache(B=B, Hkv=Hkv, D=D, n_pages=8, max_blocks=1 << 12)
            sizes = [lib.tsa_kv8_workspace_bytes(ref(c), T, Hq, 64 * nb, 0) for nb in list(range(1, 200)) + [500, 1 << 11, 1 << 12]]
            assert sizes == sorted(sizes), (D, B, Hkv, Hq, T)


def test_cache_object_refuses():
    for kw in (dict(B=0), dict(Hkv=0), dict(D=96), dict(max_len=0), dict(n_pages=0), dict(device="cpu")):
        a = dict(B=1, Hkv=1, D=64, max_len=64)
        a.update(kw)
        with pytest.raises(ValueError):
            tsa.Kv8Cache(**a)
