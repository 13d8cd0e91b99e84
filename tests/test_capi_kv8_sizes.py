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
