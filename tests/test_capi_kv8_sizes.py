"""Sizes that the 8-bit cache's entry points take or refuse, by what each of them needs (no kernel is
launched: calls that are accepted stop at their workspace)."""
import tsa
from test_capi_kv8 import attn, cache, ref, rows, select, sparse


def test_long_queries_over_a_large_capacity():
    """T times the cache's blocks passes 2^31 - 1: attention has nothing of that size; a selection has a
    score for each query and block, of max_len and not of the capacity."""
    lib = tsa.load()
    T, blocks = 300, 1 << 23
    assert T * blocks > (1 << 31) - 1
    c = cache(B=1, Hkv=1, max_blocks=blocks)
    assert lib.tsa_kv8_workspace_bytes(ref(c), T, 1, 64 * blocks, 0) > 0
    assert attn(c, T=T, Hq=1, max_len=64 * blocks, ws=None) == tsa.TSA_ERR_WORKSPACE
    assert attn(c, T=T, Hq=1, max_len=64 * blocks, q=rows(t=63)) == tsa.TSA_ERR_ARG
    assert sparse(c, T=T, Hq=1, o=rows(t=63)) == tsa.TSA_ERR_ARG
    assert lib.tsa_kv8_workspace_bytes(ref(c), T, 1, 64 * 1000, 4) >= 4 * 300 * 1000
    assert select(c, T=T, Hq=1, max_len=64 * 1000, ws=None) == tsa.TSA_ERR_WORKSPACE
    assert lib.tsa_kv8_workspace_bytes(ref(c), T, 1, 64 * blocks, 4) == 0
    assert select(c, T=T, Hq=1, max_len=64 * blocks) == tsa.TSA_ERR_SHAPE


def test_workspace_serves_shorter_lengths_where_the_tiles_change():
    """65 to 128 rows at D = 64 are cut otherwise over few blocks than over many: a workspace for the
    longer lengths still serves the shorter."""
    lib = tsa.load()
    for B, Hkv, Hq, T in ((1, 1, 1, 100), (1, 8, 8, 128), (16, 8, 32, 20), (32, 2, 16, 9), (64, 8, 8, 70), (300, 2, 16, 16)):
        c = cache(B=B, Hkv=Hkv, max_blocks=1 << 14)
        edge = 4096 // (B * Hkv)
        lengths = sorted({max(1, n) for n in [1, 2, 3, 5, 9, 17, 100, 1 << 14, *range(edge - 3, edge + 4)]})
        sizes = [lib.tsa_kv8_workspace_bytes(ref(c), T, Hq, 64 * nb, 0) for nb in lengths]
        assert sizes == sorted(sizes), (B, Hkv, Hq, T)
