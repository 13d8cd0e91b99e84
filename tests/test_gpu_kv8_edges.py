"""The 8-bit K/V cache on the GPU: uses at the edge of what its header allows, against the same
definitions and bounds as test_gpu_kv8.py."""
import math
import random

import pytest
import torch

import kv8_oracle as ko
import tsa
from test_gpu_kv8 import check_out, check_rows, expect, fill, ints, keys, rand

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------
# cutting back, again and again
# ---------------------------------------------------------------------------------------
def check_holds(c, k, v, lens, what, dev):
    """The cache's sequences are k[b], v[b] [H, len, D], bit for bit."""
    kg, vg = (x.cpu() for x in tsa.kv8_read(c, ints(lens, dev), S=max(max(lens), 1)))
    for b, n in enumerate(lens):
        for h in range(c.Hkv):
            check_rows(kg[b, h, :n], ko.Head(k[b][h, :n]).read, (what, b, h, "k"))
            check_rows(vg[b, h, :n], ko.Head(v[b][h, :n]).read, (what, b, h, "v"))


@pytest.mark.parametrize("seed", range(4))
def test_cut_back_many_times(dev, seed):
    """Writes of every size and cuts in turn, several between two writes, to any length from the lowest
    on and to whole blocks below it: each time the sequence goes on as if what was cut had never come."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(50 + seed)
    D, H, cap = (64, 128, 256, 64)[seed], 2, 640
    c = tsa.Kv8Cache(1, H, D, cap, device=dev)
    k, v, lowest = torch.zeros(H, 0, D).half(), torch.zeros(H, 0, D).half(), 0
    for i in range(14):
        T = min(rng.choice([1, 1, 2, 5, 17, 63, 64, 65, 128, 129, 200]), cap - k.shape[1])
        if T == 0:
            k, v, lowest = k[:, :64], v[:, :64], 64
            continue
        kn, vn = (x[0] for x in keys(gen, 1, H, T, D))
        k, v = torch.cat([k, kn], 1), torch.cat([v, vn], 1)
        n = k.shape[1]
        tsa.kv8_write(c, kn[None].to(dev), vn[None].to(dev), ints([n], dev))
        lowest = max(lowest, 64 * ((n - 1) // 64 - 1))
        check_holds(c, [k], [v], [n], (seed, i, "written"), dev)
        for _ in range(rng.randint(0, 2)):
            n = k.shape[1]
            n = 64 * rng.randint(0, n // 64) if rng.random() < 0.3 else rng.randint(min(lowest, n), n)
            k, v, lowest = k[:, :n], v[:, :n], min(lowest, n)
            check_holds(c, [k], [v], [n], (seed, i, "cut"), dev)
    n = k.shape[1]
    q = rand(gen, 1, 2 * H, 1, D)
    want, tol = expect(q, k[None], v[None], [n], [1], True) if n else (torch.zeros_like(q).double(), torch.zeros_like(q).double())
    check_out(tsa.attn_kv8_fwd(q.to(dev), c, ints([n], dev)).cpu(), want, tol, seed)


def test_cut_back_behind_a_shared_prefix(dev):
    """A sequence that took over 128 tokens in another's pages is cut back to no less than those, and to
    a whole block inside them with pages of its own named first: the other sequence keeps its bytes."""
    gen = torch.Generator().manual_seed(61)
    D, H = 64, 2
    k, v = keys(gen, 2, H, 360, D)
    k[1, :, :128], v[1, :, :128] = k[0, :, :128], v[0, :, :128]
    c = tsa.Kv8Cache(2, H, D, 320, n_pages=9, device=dev)
    c.table.copy_(ints([[0, 1, 2, 3, -1], [0, 1, 4, 5, 6]], dev))

    def write(at, new):
        T = max(new)
        kn, vn = (torch.stack([x[b, :, at[b]:at[b] + T] for b in range(2)]) for x in (k, v))
        tsa.kv8_write(c, kn.to(dev), vn.to(dev), ints([a + n for a, n in zip(at, new)], dev), ints(new, dev))

    write([0, 128], [128, 0])
    write([128, 128], [70, 5])
    lens = [198, 133]
    check_holds(c, k, v, lens, "written", dev)
    pages = [getattr(c, x)[:4].clone() for x in ("k", "v", "k_scale", "v_scale", "k_sum", "k_sum_scale")]
    for n, T in ((130, 60), (128, 100), (192, 7)):  # the lowest length is 128 each time
        check_holds(c, k, v, [198, n], ("cut", n), dev)
        k[1:, :, n:], v[1:, :, n:] = keys(gen, 1, H, 360 - n, D)
        write([198, n], [0, T])
        check_holds(c, k, v, [198, n + T], ("on from", n), dev)
    c.table[1, 1] = 7
    k[1:, :, 64:], v[1:, :, 64:] = keys(gen, 1, H, 296, D)
    write([198, 64], [0, 150])
    check_holds(c, k, v, [198, 214], "on from a whole block", dev)
    for x, before in zip(("k", "v", "k_scale", "v_scale", "k_sum", "k_sum_scale"), pages):
        assert torch.equal(getattr(c, x)[:4], before), x


# ---------------------------------------------------------------------------------------
# rows that see no key, infinities in open keys, output over the queries
# ---------------------------------------------------------------------------------------
FORMS = [(64, 2, 3), (128, 6, 1), (256, 1, 5), (64, 1, 40), (128, 2, 30), (256, 3, 20), (64, 3, 70), (128, 2, 170), (256, 1, 300)]


@pytest.mark.parametrize("D,G,T", FORMS)
@pytest.mark.parametrize("causal", [True, False])
def test_rows_in_front_of_the_sequence(dev, D, G, T, causal):
    """More new tokens than the sequence has: those in front of position 0 see no key, with the causal
    mask and without it, and their rows are 0; the others attend as ever."""
    gen = torch.Generator().manual_seed(D + T)
    lens, new = [max(1, T // 2), 1, 0, T], [T, T, T, T]
    B = len(lens)
    k, v = keys(gen, B, 1, T, D)
    c = tsa.Kv8Cache(B, 1, D, T, device=dev)
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints(lens, dev), ints(lens, dev))
    q = rand(gen, B, G, T, D)
    for counts in (None, ints(new, dev)):
        out = torch.full(q.shape, 9.0, dtype=torch.float16, device=dev)
        tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev), counts, out=out, causal=causal)
        for b, n in enumerate(lens):
            assert not bool(out[b, :, :T - n].any()), (b, causal)
            if n:
                want, tol = expect(q[b:b + 1, :, T - n:], k[b:b + 1], v[b:b + 1], [n], [n], causal)
                check_out(out[b:b + 1, :, T - n:].cpu(), want, tol, (b, causal))


@pytest.mark.parametrize("D,G,T", FORMS)
@pytest.mark.parametrize("what", [math.inf, -math.inf])
def test_infinite_key_in_the_open_block(dev, D, G, T, what):
    """A query's score with it is an infinity of its own sign: below every other, the key weighs 0 and
    the rest stays; above them, the row is NaN.  Queries in front of it see neither."""
    gen = torch.Generator().manual_seed(D + G + T)
    L = 64 * max(3, T // 64 + 1) + 40
    where = L - 1 - T // 2 if T < 40 else L - 20
    k, v = keys(gen, 1, 1, L, D)
    q = rand(gen, 1, G, T, D)
    q[..., 5] = torch.where(q[..., 5] < 0, -1, 1) * q[..., 5].abs().clamp_min(0.01)
    k[0, 0, where, 5] = what
    o = tsa.attn_kv8_fwd(q.to(dev), fill(dev, k, v, [L]), ints([L], dev)).cpu()
    k[0, 0, where, 5] = 0
    K, V = ko.Head(k[0, 0]).values, ko.Head(v[0, 0])
    for g in range(G):
        for t in range(T):
            p = L - T + t
            if p >= where and float(q[0, g, t, 5]) * what > 0:
                assert bool(o[0, g, t].isnan().all()), (g, t)
            else:
                see = [j for j in range(p + 1) if j != where]
                want, tol = ko.attend(q[0, g, t], K, V.values, V.steps, see, 1 / math.sqrt(D))
                check_out(o[0, g, t], want, tol, (g, t))


@pytest.mark.parametrize("D,G,T", FORMS)
def test_output_over_the_queries(dev, D, G, T):
    """o = q in every form, its keys split or not: the same bytes as in a buffer of its own."""
    gen = torch.Generator().manual_seed(2 * D + T)
    for H, L in ((2, T + 70), (1, T + 2500)):
        k, v = (x.to(dev) for x in keys(gen, 2, H, L, D))
        n = ints([L, L - 50], dev)
        c = tsa.Kv8Cache(2, H, D, L, device=dev)
        tsa.kv8_write(c, k, v, n, n)
        buf = rand(gen, 2, T, H * G, 2 * D).to(dev)  # a token-major projection of q and gate
        q, gate = buf[..., :D].transpose(1, 2), buf[..., D:].transpose(1, 2)
        blocks = tsa.kv8_select(q, c, n, 4)
        for call in (lambda **kw: tsa.attn_kv8_fwd(q, c, n, gate=gate, **kw), lambda **kw: tsa.attn_kv8_blocks_fwd(q, c, n, blocks, gate=gate, **kw)):
            before = q.clone()
            want = call()
            call(out=q)
            assert torch.equal(q, want), (H, L)
            q.copy_(before)


def test_output_over_the_queries_of_many_listed_tiles(dev):
    """The form that takes a listed tile a wave, and a group of more heads than a tile has."""
    gen = torch.Generator().manual_seed(71)
    D, H, G, T, L = 64, 2, 17, 600, 900
    k, v = (x.to(dev) for x in keys(gen, 1, H, L, D))
    n = ints([L], dev)
    c = tsa.Kv8Cache(1, H, D, L, device=dev)
    tsa.kv8_write(c, k, v, n)
    q = rand(gen, 1, H * G, T, D).to(dev)
    blocks = tsa.kv8_select(q, c, n, 3)
    want = tsa.attn_kv8_blocks_fwd(q, c, n, blocks)
    tsa.attn_kv8_blocks_fwd(q, c, n, blocks, out=q)
    assert torch.equal(q, want)


@pytest.mark.parametrize("D,T", [(64, 300), (128, 260)])
def test_long_queries_over_a_large_capacity(dev, D, T):
    """Queries and blocks of capacity whose product passes 32 bits, with a few blocks in use; a selection
    with a max_len that holds every sequence."""
    gen = torch.Generator().manual_seed(81)
    L = T + 150
    k, v = keys(gen, 1, 1, L, D)
    c = tsa.Kv8Cache(1, 1, D, 64 << 23, n_pages=8, device=dev)
    c.table[0, :8] = torch.arange(8, dtype=torch.int32, device=dev)
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints([L], dev))
    q = rand(gen, 1, 1, T, D)
    want, tol = expect(q, k, v, [L], [T], True)
    check_out(tsa.attn_kv8_fwd(q.to(dev), c, ints([L], dev)).cpu(), want, tol, "dense")
    blocks = tsa.kv8_select(q.to(dev), c, ints([L], dev), 100, max_len=L)
    check_out(tsa.attn_kv8_blocks_fwd(q.to(dev), c, ints([L], dev), blocks).cpu(), want, tol, "sparse")
    with pytest.raises(tsa.TsaError) as e:
        tsa.kv8_select(q.to(dev), c, ints([L], dev), 100)
    assert e.value.code == tsa.TSA_ERR_SHAPE


@pytest.mark.parametrize("G,T", [(1, 65), (2, 40), (8, 16), (4, 32)])
@pytest.mark.parametrize("blocks", [64, 4096, 4097])
def test_tiles_of_medium_row_counts(dev, G, T, blocks):
    """65 to 128 rows at D = 64: two tiles of 64 rows, and with max_len behind 4096 blocks one of 128."""
    gen = torch.Generator().manual_seed(90 + T)
    lens = [T + 777]
    k, v = keys(gen, 1, 1, lens[0], 64)
    c = tsa.Kv8Cache(1, 1, 64, 64 * blocks, device=dev)
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints(lens, dev))
    q = rand(gen, 1, G, T, 64)
    o = tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev))
    want, tol = expect(q, k, v, lens, [T], True)
    check_out(o.cpu(), want, tol, (G, T, blocks))


def test_numbers_beyond_32_bits(dev):
    """A max_len behind any length is the cache's own; numbers of blocks that no C int holds are refused."""
    gen = torch.Generator().manual_seed(95)
    D, L = 64, 64 * 20 + 5
    k, v = keys(gen, 1, 1, L, D)
    c = fill(dev, k, v, [L])
    q, n = rand(gen, 1, 2, 3, D).to(dev), ints([L], dev)
    for far in (1 << 31, (1 << 32) + 64, 1 << 40):
        assert tsa.kv8_workspace_bytes(c, 3, 2, far) == tsa.kv8_workspace_bytes(c, 3, 2)
        assert torch.equal(tsa.attn_kv8_fwd(q, c, n, max_len=far), tsa.attn_kv8_fwd(q, c, n))
        assert torch.equal(tsa.kv8_select(q, c, n, 5, max_len=far), tsa.kv8_select(q, c, n, 5))
        for kw in (dict(first=far), dict(recent=far), dict(first=-far - 1)):
            with pytest.raises(ValueError):
                tsa.kv8_select(q, c, n, 5, **kw)


@pytest.mark.parametrize("D,B,Hkv,G,T,L,cap", [(64, 1, 2, 4, 1, 3000, 3000), (128, 5, 2, 3, 2, 700, 1 << 16), (256, 1, 4, 6, 1, 500, 1 << 15), (64, 70, 1, 2, 1, 200, 1 << 14),
                                               (64, 2, 1, 8, 9, 900, 900), (64, 1, 1, 8, 70, 2000, 2000), (128, 1, 2, 2, 40, 1500, 1500), (256, 1, 1, 1, 300, 2500, 2500)])
def test_workspace_of_exactly_its_size(dev, D, B, Hkv, G, T, L, cap):
    """A call keeps within the bytes that it asks for, with max_len exact, too short and as large as the
    cache, and gives the same rows whatever the workspace held."""
    gen = torch.Generator().manual_seed(D + T)
    c = tsa.Kv8Cache(B, Hkv, D, cap, n_pages=B * (L // 64 + 1), device=dev)
    c.table[:, :L // 64 + 1] = torch.arange(c.n_pages, dtype=torch.int32, device=dev).view(B, -1)
    k, v = (rand(gen, B, Hkv, L, D).to(dev) for _ in range(2))
    n = ints([L - 3 * b for b in range(B)], dev)
    tsa.kv8_write(c, k, v, n, n)
    q = rand(gen, B, Hkv * G, T, D).to(dev)

    def guarded(bytes_, fill_):
        ws = torch.full((bytes_ + 4096,), fill_, dtype=torch.uint8, device=dev)
        return ws, ws[:bytes_]

    for max_len in (L, 64, None):
        outs = []
        for byte in (0xff, 0):
            whole, ws = guarded(tsa.kv8_workspace_bytes(c, T, Hkv * G, max_len), byte)
            outs.append(tsa.attn_kv8_fwd(q, c, n, max_len=max_len, ws=ws))
            assert bool((whole[len(ws):] == byte).all())
        assert torch.equal(*outs)
    outs = []
    for byte in (0xff, 0):
        whole, ws = guarded(tsa.kv8_workspace_bytes(c, T, Hkv * G, L, 4), byte)
        blocks = tsa.kv8_select(q, c, n, 4, max_len=L, ws=ws)
        outs.append((blocks, tsa.attn_kv8_blocks_fwd(q, c, n, blocks, ws=ws)))
        assert bool((whole[len(ws):] == byte).all())
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("D,G,T", FORMS)
def test_scores_of_minus_infinity_alone(dev, D, G, T):
    """Every key that the first rows see is minus infinity in a channel where q is positive: their
    scores leave nothing to weigh, and they are 0; the other rows go on without those keys."""
    gen = torch.Generator().manual_seed(3 * D + T)
    T = min(T, 60)
    k, v = keys(gen, 1, 1, T, D)
    q = rand(gen, 1, G, T, D)
    q[..., 5] = q[..., 5].abs().clamp_min(0.01)
    first = (T + 1) // 2
    k[0, 0, :first, 5] = -math.inf
    o = tsa.attn_kv8_fwd(q.to(dev), fill(dev, k, v, [T]), ints([T], dev)).cpu()
    assert not bool(o[:, :, :first].any())
    K, V = k[0, 0, first:].double(), v[0, 0, first:].double()
    for g in range(G):
        for t in range(first, T):
            want, tol = ko.attend(q[0, g, t], K, V, torch.ones(T - first, dtype=torch.float64), list(range(t - first + 1)), 1 / math.sqrt(D))
            check_out(o[0, g, t], want, tol, (g, t))
