"""The 8-bit K/V cache on the GPU: written, read back, attended to and selected from, against the
definitions in 64 bits (kv8_oracle.py).  Codes, scales, summaries, read-back values and selected
blocks are equal bit for bit; attention within the bound that kv8_oracle.attend derives."""
import math

import numpy as np
import pytest
import torch

import kv8_oracle as ko
import tsa

pytestmark = pytest.mark.gpu


def rand(gen, *shape):
    return torch.randn(*shape, generator=gen).half()


def keys(gen, B, H, L, D):
    """K, V [B, H, L, D] fp16 on the CPU: channels of unequal size, blocks with a mean of their own."""
    k = rand(gen, B, H, L, D).float() * torch.exp(0.5 * torch.randn(1, H, 1, D, generator=gen))
    nb = -(-L // 64)
    k += torch.randn(B, H, nb, 1, D, generator=gen).expand(B, H, nb, 64, D).reshape(B, H, nb * 64, D)[:, :, :L]
    return k.half(), rand(gen, B, H, L, D)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def fill(dev, k, v, lens, max_len=None, **kw):
    """A cache that holds the first lens[b] rows of k, v."""
    B, H, L, D = k.shape
    c = tsa.Kv8Cache(B, H, D, max_len or L, device=dev, **kw)
    if L and max(lens):
        tsa.kv8_write(c, k.to(dev), v.to(dev), ints(lens, dev), ints(lens, dev))
    return c


def check_rows(got, want, what):
    assert got.dtype == want.dtype == torch.float16
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool(same.all()), (what, int((~same).sum()), got[~same][:4], want[~same][:4])


def check_out(got, want, tol, what):
    """got fp16, want and tol in 64 bits; a NaN or infinity only where the definition has it."""
    got = got.double()
    fine = torch.isfinite(want)
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), what
    assert bool((got[~fine & ~want.isnan()] == want[~fine & ~want.isnan()]).all()), what
    off = (got - want).abs()[fine] - tol[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - want).abs()[fine].max()))


def expect(q, k, v, lens, n_new, causal, gate=None, scale=None, lists=None, pages=None):
    """The output and its bound for q [B, Hq, T, D] over k, v [B, H, L, D]; rows of padding are NaN."""
    B, Hq, T, D = q.shape
    H = k.shape[1]
    G = Hq // H
    want = torch.full(q.shape, math.nan, dtype=torch.float64)
    tol = torch.zeros_like(want)
    scale = scale or 1 / math.sqrt(D)
    for b in range(B):
        n, L = n_new[b], lens[b]
        for h in range(H):
            K, V = ko.Head(k[b, h, :L]).values, ko.Head(v[b, h, :L])
            for t in range(n):
                p = L - n + t
                see = list(range(p + 1 if causal else L)) if p >= 0 or not causal else []
                if lists is not None:
                    see = [j for blk in lists[b][h][t] if 0 <= blk <= max(p, -1) // 64 for j in range(blk * 64, min(blk * 64 + 64, p + 1))]
                if pages is not None:
                    see = [j for j in see if pages[b][j // 64] or j >= L // 64 * 64]
                for g in range(G):
                    hq = h * G + g
                    want[b, hq, t], tol[b, hq, t] = ko.attend(q[b, hq, t], K, V.values, V.steps, see, scale, None if gate is None else gate[b, hq, t])
    return want, tol


# ---------------------------------------------------------------------------------------
# write and read
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cuts", [[200], [1] * 70, [64, 64], [63, 1, 1], [5, 60, 130, 1], [128, 7, 200, 64], [1, 300]],
                         ids=lambda c: "70x1" if len(c) == 70 else "+".join(map(str, c)))
def test_write_and_read_back(dev, D, cuts):
    gen = torch.Generator().manual_seed(D + len(cuts))
    H, L = 2, sum(cuts)
    k, v = keys(gen, 1, H, L, D)
    c = tsa.Kv8Cache(1, H, D, L + 64, device=dev)
    n = 0
    for T in cuts:
        tsa.kv8_write(c, k[:, :, n:n + T].contiguous().to(dev), v[:, :, n:n + T].contiguous().to(dev), ints([n + T], dev))
        n += T
    kg, vg = tsa.kv8_read(c, ints([L], dev))
    for h in range(H):
        for x, got, scales in ((k, kg, c.k_scale), (v, vg, c.v_scale)):
            head = ko.Head(x[0, h])
            check_rows(got[0, h, :L].cpu(), head.read, (D, cuts, h))
            assert scales[:L // 64, h].cpu().tolist() == head.scales
            assert not bool(got[0, h, L:].any())
            for i in range(L // 64) if x is k else ():
                m, s = head.summary(i)
                assert torch.equal(c.k_sum[i, h].cpu().double(), m)
                assert c.k_sum_scale[i, h].item() == float(s)


def test_how_tokens_come_does_not_matter(dev):
    """One call, single tokens and uneven pieces leave the same cache, every byte of it that holds tokens."""
    gen = torch.Generator().manual_seed(3)
    D, H, L = 128, 3, 64 * 5 + 33
    k, v = (x.to(dev) for x in keys(gen, 1, H, L, D))
    caches = []
    for cuts in ([L], [1] * L, [100, 1, 27, 129, 64, L - 321]):
        c, n = tsa.Kv8Cache(1, H, D, L, device=dev), 0
        for T in cuts:
            tsa.kv8_write(c, k[:, :, n:n + T], v[:, :, n:n + T], ints([n + T], dev))
            n += T
        caches.append(c)
    for c in caches[1:]:
        for name in ("k", "v", "k_scale", "v_scale", "k_sum", "k_sum_scale"):
            assert torch.equal(getattr(c, name), getattr(caches[0], name)), name
        # the ring: block 4's rows whole, and of block 5's the 33 that there are (behind them lies
        # what block 3 left, or nothing)
        assert torch.equal(c.k_open[:, 0], caches[0].k_open[:, 0]) and torch.equal(c.v_open[:, 0], caches[0].v_open[:, 0])
        for x, y in zip(tsa.kv8_read(c, ints([L], dev)), tsa.kv8_read(caches[0], ints([L], dev))):
            assert torch.equal(x, y)


def test_write_ragged_and_padded(dev):
    """Sequences of 0, 1, 63, 64, 65 and 130 new tokens in one padded call, on top of what is there;
    the padding holds NaN and is not looked at, the slots without new tokens keep theirs."""
    gen = torch.Generator().manual_seed(5)
    D, H, T = 64, 2, 130
    old, new = [10, 0, 64, 1, 63, 70], [0, 1, 63, 64, 65, 130]
    B = len(old)
    k, v = keys(gen, B, H, 200, D)
    c = fill(dev, k, v, old)
    kn, vn = (torch.full((B, H, T, D), math.nan).half() for _ in range(2))
    for b in range(B):
        kn[b, :, :new[b]] = k[b, :, old[b]:old[b] + new[b]]
        vn[b, :, :new[b]] = v[b, :, old[b]:old[b] + new[b]]
    lens = [o + n for o, n in zip(old, new)]
    tsa.kv8_write(c, kn.to(dev), vn.to(dev), ints(lens, dev), ints(new, dev))
    ko_, vo_ = (torch.full((B, H, 200, D), 7.0, dtype=torch.float16, device=dev) for _ in range(2))
    tsa.kv8_read(c, ints(lens, dev), k_out=ko_, v_out=vo_)
    for b in range(B):
        for h in range(H):
            for x, got in ((k, ko_), (v, vo_)):
                check_rows(got[b, h, :lens[b]].cpu(), ko.Head(x[b, h, :lens[b]]).read, (b, h))
                assert bool((got[b, h, lens[b]:] == 7).all())


def test_counts_out_of_range(dev):
    """More new tokens than the sequence has: those in front of it are dropped.  A length behind the
    cache's end, negative lengths and counts: taken as the nearest that is possible."""
    gen = torch.Generator().manual_seed(6)
    D, H = 64, 1
    k, v = keys(gen, 4, H, 128, D)
    c = tsa.Kv8Cache(4, H, D, 128, device=dev)
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints([50, -3, 1000, 128], dev), ints([90, 5, 128, -1], dev))
    kg, _ = tsa.kv8_read(c, ints([50, 0, 999, 0], dev))
    check_rows(kg[0, 0, :50].cpu(), k[0, 0, 40:90], "dropped")
    check_rows(kg[2, 0].cpu(), ko.Head(k[2, 0]).read, "to the end")
    assert not bool(kg[[1, 3]].any())
    q = rand(gen, 4, H, 90, D)
    o = tsa.attn_kv8_fwd(q.to(dev), c, ints([50, -3, 1000, 128], dev), ints([90, 5, 0, -1], dev)).cpu()
    assert not bool(o[0, :, :40].any()) and not bool(o[1:].any())
    want, tol = expect(q[:1, :, 40:], k[:1, :, 40:90], v[:1, :, 40:90], [50], [50], True)
    check_out(o[:1, :, 40:], want, tol, "behind the front")


def test_read_ranges_and_strides(dev):
    gen = torch.Generator().manual_seed(7)
    D, H, B = 128, 2, 3
    lens = [300, 65, 200]
    k, v = keys(gen, B, H, 300, D)
    c = fill(dev, k, v, lens)
    start = [37, 64, 500]
    out = torch.full((B, 100, H, 2, D), 5.0, dtype=torch.float16, device=dev)  # token-major, between others
    view = out[:, :, :, 1].transpose(1, 2)
    got, none = tsa.kv8_read(c, ints(lens, dev), start=ints(start, dev), k_out=view)
    assert none is None
    for b in range(B):
        n = max(0, min(100, lens[b] - start[b]))
        for h in range(H):
            check_rows(view[b, h, :n].cpu(), ko.Head(k[b, h, :lens[b]]).read[start[b]:start[b] + n], (b, h))
            assert bool((view[b, h, n:] == 5).all())
    assert bool((out[:, :, :, 0] == 5).all())


def test_write_from_strided_rows(dev):
    """Keys and values as slices of one token-major projection, and rows broadcast over heads."""
    gen = torch.Generator().manual_seed(8)
    D, H, T = 64, 2, 150
    proj = rand(gen, 1, T, 2 * H + 3, D).to(dev)
    k, v = proj[:, :, 1:1 + H].transpose(1, 2), proj[:, :, 2 + H:2 + H + 1].transpose(1, 2).expand(1, H, T, D)
    c = tsa.Kv8Cache(1, H, D, T, device=dev)
    tsa.kv8_write(c, k, v, ints([T], dev))
    kg, vg = tsa.kv8_read(c, ints([T], dev), S=T)
    for h in range(H):
        check_rows(kg[0, h].cpu(), ko.Head(k[0, h].cpu()).read, h)
        check_rows(vg[0, h].cpu(), ko.Head(v[0, h].cpu()).read, h)


def test_ties_and_extremes(dev):
    """Codes halfway between two (x = a / 2 and its like), the smallest and largest fp16, zeros."""
    D = 64
    x = torch.zeros(5 * 64, D).half()
    x[:64] = torch.arange(-127, 127).repeat(17)[:64 * D].view(64, D).half() * 0.5  # a = 63.5, ties
    x[64:128] = torch.tensor([65504.0, -65504.0, 32752.0, 6e-8] * 16).half()
    x[128:192] = 0
    x[192:256] = 2.0 ** -24
    x[256:] = torch.linspace(-254, 254, 64 * D).view(64, D).half()
    c = tsa.Kv8Cache(1, 1, D, 320, device=dev)
    xd = x.view(1, 1, 320, D).to(dev)
    tsa.kv8_write(c, xd, xd, ints([320], dev))
    kg, vg = tsa.kv8_read(c, ints([320], dev))
    head = ko.Head(x)
    check_rows(kg[0, 0].cpu(), head.read, "k")
    check_rows(vg[0, 0].cpu(), head.read, "v")
    for i in range(5):
        assert torch.equal(c.k_sum[i, 0].cpu().double(), head.summary(i)[0])


def test_cut_back(dev):
    """A sequence cut back by up to a block of tokens, across a block's end, goes on as if they had never come."""
    gen = torch.Generator().manual_seed(9)
    D, H = 128, 2
    for length, back in ((130, 10), (128, 64), (200, 64), (64, 1)):
        k, v = keys(gen, 1, H, length + 40, D)
        c = fill(dev, k, v, [length], max_len=320)
        n = length - back
        k2, v2 = keys(gen, 1, H, length + 40, D)
        k2[:, :, :n], v2[:, :, :n] = k[:, :, :n], v[:, :, :n]
        kg, _ = tsa.kv8_read(c, ints([n], dev), S=n if n else 1)
        if n:
            check_rows(kg[0, 0].cpu(), ko.Head(k[0, 0, :n]).read, (length, back))
        T = length + 40 - n
        tsa.kv8_write(c, k2[:, :, n:].to(dev), v2[:, :, n:].to(dev), ints([n + T], dev))
        kg, vg = tsa.kv8_read(c, ints([n + T], dev), S=n + T)
        for h in range(H):
            check_rows(kg[0, h].cpu(), ko.Head(k2[0, h]).read, (length, back, h))
            check_rows(vg[0, h].cpu(), ko.Head(v2[0, h]).read, (length, back, h))


def test_pages(dev):
    """Pages in any order, full blocks shared by two sequences, blocks without a page and numbers that
    are none: nothing of theirs is written, and no query sees their keys."""
    gen = torch.Generator().manual_seed(10)
    D, H, L = 64, 2, 64 * 4 + 20
    k, v = keys(gen, 3, H, L, D)
    k[1, :, :128], v[1, :, :128] = k[0, :, :128], v[0, :, :128]
    c = tsa.Kv8Cache(3, H, D, L, n_pages=9, device=dev)
    assert bool((c.table == -1).all())
    c.table.copy_(ints([[8, 2, 5, 0, 7], [8, 2, 1, 6, 7], [3, -1, 4, 9, 1 << 30]], dev))
    before = c.k[7].clone()
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints([L] * 3, dev))
    assert torch.equal(c.k[7], before)
    kg, _ = tsa.kv8_read(c, ints([L] * 3, dev))
    for b in range(3):
        want = ko.Head(k[b, 1]).read.clone()
        if b == 2:
            want[64:128] = 0
            want[192:256] = 0
        check_rows(kg[b, 1, :L].cpu(), want, b)
    q = rand(gen, 3, 2 * H, 2, D)
    o = tsa.attn_kv8_fwd(q.to(dev), c, ints([L] * 3, dev))
    pages = [[True] * 5, [True] * 5, [True, False, True, False, False]]
    want, tol = expect(q, k, v, [L] * 3, [2] * 3, True, pages=pages)
    check_out(o.cpu(), want, tol, "pages")
    # only blocks without a page, and no open one: rows that see nothing
    c.table[0].fill_(-1)
    o = tsa.attn_kv8_fwd(q.to(dev), c, ints([256, L, L], dev))
    assert not bool(o[0].any())
    o = tsa.attn_kv8_blocks_fwd(q.to(dev), c, ints([256, L, L], dev), ints([0, 1, 2], dev).expand(3, H, 2, 3).contiguous())
    assert not bool(o[0].any())


def test_offsets_beyond_32_bits(dev):
    """Pages behind the 4 GiB of codes that 32-bit offsets reach, next to low ones."""
    gen = torch.Generator().manual_seed(11)
    D, H, L = 256, 1, 64 * 3 + 5
    n_pages = (1 << 32) // (64 * D) + 10
    k, v = keys(gen, 1, H, L, D)
    c = tsa.Kv8Cache(1, H, D, L, n_pages=n_pages, device=dev)
    c.table.copy_(ints([[n_pages - 1, 3, n_pages - 7, 0]], dev))
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints([L], dev))
    kg, vg = tsa.kv8_read(c, ints([L], dev), S=L)
    check_rows(kg[0, 0].cpu(), ko.Head(k[0, 0]).read, "k")
    check_rows(vg[0, 0].cpu(), ko.Head(v[0, 0]).read, "v")
    q = rand(gen, 1, 6, 1, D)
    want, tol = expect(q, k, v, [L], [1], True)
    check_out(tsa.attn_kv8_fwd(q.to(dev), c, ints([L], dev)).cpu(), want, tol, "far pages")


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G,T", [(1, 1), (6, 1), (17, 1), (3, 2), (8, 5), (2, 33), (1, 70), (3, 131)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(dev, D, G, T, causal):
    gen = torch.Generator().manual_seed(100 * D + 10 * G + T)
    H = 2
    lens = [max(n, T) for n in (T, 1, 63, 64, 65, 200, 321)]
    B = len(lens)
    k, v = keys(gen, B, H, max(lens), D)
    c = fill(dev, k, v, lens)
    q, gate = rand(gen, B, H * G, T, D), rand(gen, B, H * G, T, D) if T % 2 else None
    o = tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev), gate=None if gate is None else gate.to(dev), causal=causal)
    want, tol = expect(q, k, v, lens, [T] * B, causal, gate)
    check_out(o.cpu(), want, tol, (D, G, T, causal))


@pytest.mark.parametrize("D,G,T,length", [(64, 2, 1, 5000), (128, 8, 1, 3333), (256, 6, 1, 4097), (128, 1, 3, 2048), (256, 6, 40, 1500)])
def test_attention_over_long_caches(dev, D, G, T, length):
    """The keys of a row are split over workgroups; whatever max_len says, the results are right."""
    gen = torch.Generator().manual_seed(length)
    lens = [length, 100 + T]
    k, v = keys(gen, 2, 1, length, D)
    c = fill(dev, k, v, lens)
    q = rand(gen, 2, G, T, D)
    want, tol = expect(q, k, v, lens, [T] * 2, True)
    for max_len in (None, 64, 1000):
        o = tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev), max_len=max_len)
        check_out(o.cpu(), want, tol, max_len)


@pytest.mark.parametrize("D,H,G,T,lens", [
    (64, 1, 2, 2, [(37 * b) % 401 for b in range(70)]),
    (128, 2, 3, 1, [64, 1, 1300, 63, 0, 65, 128, 700]),
    (256, 3, 2, 3, [900, 5, 0, 64, 1500]),
    (256, 1, 6, 1, [2500, 2500, 2500]),
    (64, 1, 2, 1, [70000, 100, 3]),
], ids=["70", "8", "5", "3", "long"])
def test_attention_over_sequences_of_a_large_cache(dev, D, H, G, T, lens):
    """A cache that could hold much more: all sequences' keys are dealt out to the workgroups, whose
    segments end anywhere and pass over sequences that are empty or without new tokens."""
    gen = torch.Generator().manual_seed(D + len(lens))
    B = len(lens)
    new = [0 if b % 5 == 3 else T - (b % 7 == 2 and T > 1) for b in range(B)]
    k, v = keys(gen, B, H, max(lens), D)
    c, page = tsa.Kv8Cache(B, H, D, 1 << 18, n_pages=sum(n // 64 for n in lens) + 1, device=dev), 0
    for b, n in enumerate(lens):
        c.table[b, :n // 64] = torch.arange(page, page + n // 64, dtype=torch.int32, device=dev)
        page += n // 64
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints(lens, dev), ints(lens, dev))
    q, gate = rand(gen, B, H * G, T, D), rand(gen, B, H * G, T, D)
    out = torch.full(q.shape, 9.0, dtype=torch.float16, device=dev)
    tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev), ints(new, dev), gate=gate.to(dev), out=out)
    want, tol = expect(q, k, v, lens, new, True, gate)
    for b in range(B):
        assert bool((out[b, :, new[b]:] == 9).all())
        check_out(out[b, :, :new[b]].cpu(), want[b, :, :new[b]], tol[b, :, :new[b]], b)


def test_attention_ragged_and_padded(dev):
    """A padded batch: rows of padding stay as they were, slots without new tokens are untouched."""
    gen = torch.Generator().manual_seed(21)
    D, H, G, T = 128, 2, 3, 20
    lens, new = [300, 20, 64, 5, 130], [0, 20, 1, 5, 13]
    B = len(lens)
    k, v = keys(gen, B, H, 300, D)
    c = fill(dev, k, v, lens)
    q = rand(gen, B, H * G, T, D)
    for b in range(B):
        q[b, :, new[b]:] = math.nan
    out = torch.full(q.shape, 9.0, dtype=torch.float16, device=dev)
    tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev), ints(new, dev), out=out)
    want, tol = expect(q, k, v, lens, new, True)
    for b in range(B):
        assert bool((out[b, :, new[b]:] == 9).all())
        check_out(out[b, :, :new[b]].cpu(), want[b, :, :new[b]], tol[b, :, :new[b]], b)


def test_attention_strides_and_in_place(dev):
    gen = torch.Generator().manual_seed(22)
    D, H, G, T, L = 64, 2, 2, 7, 150
    k, v = keys(gen, 1, H, L, D)
    c = fill(dev, k, v, [L])
    buf = rand(gen, 1, T, H * G, 2 * D).to(dev)  # a token-major projection of q and gate
    q, gate = buf[..., :D].transpose(1, 2), buf[..., D:].transpose(1, 2)
    want, tol = expect(q.cpu(), k, v, [L], [T], True, gate.cpu())
    out = torch.zeros(1, T, H * G, D, dtype=torch.float16, device=dev).transpose(1, 2)
    tsa.attn_kv8_fwd(q, c, ints([L], dev), gate=gate, out=out)
    check_out(out.cpu(), want, tol, "strides")
    tsa.attn_kv8_fwd(q, c, ints([L], dev), gate=gate, out=q)
    check_out(q.cpu(), want, tol, "in place")


@pytest.mark.parametrize("T", [1, 6, 90])
def test_unequal_block_scales(dev, T):
    """Blocks of values 2^20 apart, the large ones far down the softmax or at its top, and blocks of
    zeros: each key counts by its weight, whatever its block's scale is."""
    gen = torch.Generator().manual_seed(23)
    D, L = 128, 64 * 6 + 10
    k, v = keys(gen, 1, 1, L, D)
    v = v.float()
    for i, f in enumerate((1.0, 2.0 ** 12, 2.0 ** -10, 0.0, 2.0 ** -14, 1.0)):
        v[:, :, 64 * i:64 * i + 64] *= f
    v = v.half()
    c = fill(dev, k, v, [L])
    q = rand(gen, 1, 4, T, D)
    for scale in (0.02, 1 / math.sqrt(D), 1.5):
        o = tsa.attn_kv8_fwd(q.to(dev), c, ints([L], dev), scale=scale)
        want, tol = expect(q, k, v, [L], [T], True, scale=scale)
        check_out(o.cpu(), want, tol, scale)


@pytest.mark.parametrize("T", [3, 80])
def test_not_finite_behind_the_mask(dev, T):
    """Infinities and NaN in keys and values of later tokens reach only the queries that see them; a
    full block that holds one is NaN as a whole."""
    gen = torch.Generator().manual_seed(24)
    D, G, L = 64, 2, 64 * 2 + 40
    for where, blocky in ((L - 1, False), (130, False), (127, True)):
        for what in (math.inf, -math.inf, math.nan):
            for side in "kv":
                k, v = keys(gen, 1, 1, L, D)
                (k if side == "k" else v)[0, 0, where, 5] = what
                c = fill(dev, k, v, [L])
                q = rand(gen, 1, G, T, D)
                o = tsa.attn_kv8_fwd(q.to(dev), c, ints([L], dev)).cpu()
                first = 64 if blocky else where  # the first key that is spoilt
                kk, vv = k.clone(), v.clone()
                (kk if side == "k" else vv)[0, 0, where, 5] = 0
                if blocky:  # the block's own values do not matter below: nothing finite sees them
                    (kk if side == "k" else vv)[0, 0, 64:128] = 0
                want, tol = expect(q, kk, vv, [L], [T], True)
                for t in range(T):
                    if L - T + t < first:
                        check_out(o[:, :, t], want[:, :, t], tol[:, :, t], (where, what, side, t))
                    elif side == "v" and not blocky:
                        bad = o[:, :, t, 5]
                        assert bool((bad.isnan() if what != what else bad == what).all()), (where, what, t)
                        for d in (4, 6):
                            check_out(o[:, :, t, d], want[:, :, t, d], tol[:, :, t, d], (where, what, side, t, d))
                    elif blocky or what != what:
                        assert bool(o[:, :, t].isnan().all()), (where, what, side, t)


@pytest.mark.parametrize("D,T", [(128, 30), (128, 150), (256, 50), (256, 150)])
def test_not_finite_behind_the_mask_of_many_rows(dev, D, T):
    """The same for two heads of T tokens, whose rows share tiles with rows that see the bad key: an open
    key's infinity and NaN, and a full block that holds one."""
    gen = torch.Generator().manual_seed(D + T)
    L = 64 * 3 + 40
    for where, what, side in ((L - 3, math.nan, "k"), (L - 3, math.nan, "v"), (L - 3, -math.inf, "v"), (190, math.inf, "k"), (190, math.nan, "v")):
        k, v = keys(gen, 1, 1, L, D)
        q = rand(gen, 1, 2, T, D)
        x = k if side == "k" else v
        x[0, 0, where, 5] = what
        o = tsa.attn_kv8_fwd(q.to(dev), fill(dev, k, v, [L]), ints([L], dev)).cpu()
        first = where if where >= 192 else 128
        x[0, 0, where, 5] = 0
        if where < 192:
            x[0, 0, 128:192] = 0
        want, tol = expect(q, k, v, [L], [T], True)
        clean = max(0, min(T, first - (L - T)))  # queries in front of the first bad key
        check_out(o[:, :, :clean], want[:, :, :clean], tol[:, :, :clean], (where, what, side))
        bad = o[:, :, clean:]
        if side == "v" and where >= 192:
            assert bool((bad[..., 5].isnan() if what != what else bad[..., 5] == what).all()), (where, what)
            for d in (4, 6):
                check_out(bad[..., d], want[:, :, clean:, d], tol[:, :, clean:, d], (where, what, d))
        else:
            assert bool(bad.isnan().all()), (where, what, side)


@pytest.mark.parametrize("D,G,T", [(64, 2, 4), (64, 1, 100), (128, 1, 40), (128, 2, 140), (256, 1, 3), (256, 2, 140)])
def test_scores_that_underflow(dev, D, G, T):
    """A scale so small that its product with a block's step is 0: every key that a query sees weighs
    the same, and one that it does not see nothing."""
    gen = torch.Generator().manual_seed(D + T)
    L = 64 * 3 + 30
    k, v = rand(gen, 1, 1, L, D) * 2.0 ** -20, rand(gen, 1, 1, L, D)
    c = fill(dev, k, v, [L])
    q = rand(gen, 1, G, T, D)
    want, tol = expect(q, k, v, [L], [T], True, scale=1e-40)
    check_out(tsa.attn_kv8_fwd(q.to(dev), c, ints([L], dev), scale=1e-40).cpu(), want, tol, (D, G, T))


def test_garbage_behind_the_sequence(dev):
    """What the ring and pages hold behind a sequence (here NaN) is not looked at."""
    gen = torch.Generator().manual_seed(25)
    D, H, lens = 128, 1, [1, 64, 100, 191]
    k, v = keys(gen, 4, H, 192, D)
    c = tsa.Kv8Cache(4, H, D, 256, device=dev)
    for t in (c.k_open, c.v_open, c.k_scale, c.v_scale, c.k_sum_scale):
        t.fill_(math.nan)
    tsa.kv8_write(c, k.to(dev), v.to(dev), ints(lens, dev), ints(lens, dev))
    q = rand(gen, 4, 3, 1, D)
    want, tol = expect(q, k, v, lens, [1] * 4, True)
    check_out(tsa.attn_kv8_fwd(q.to(dev), c, ints(lens, dev)).cpu(), want, tol, "garbage")


# ---------------------------------------------------------------------------------------
# selection and attention over selected blocks
# ---------------------------------------------------------------------------------------
def chosen(q, k, lens, n_new, top, first, recent, **kw):
    B, Hq, T, _ = q.shape
    H = k.shape[1]
    G = Hq // H
    heads = [[ko.Head(k[b, h, :lens[b]]) for h in range(H)] for b in range(B)]
    return [[[ko.select(q[b, h * G:(h + 1) * G, t], heads[b][h], lens[b] - n_new[b] + t, top, first, recent, **kw)
              for t in range(n_new[b])] for h in range(H)] for b in range(B)]


def as_lists(blocks):
    """The lists of a selection; each has to be filled from the front, -1 behind."""
    out = []
    for x in blocks.cpu().flatten(0, 2).tolist():
        n = sum(i >= 0 for i in x)
        assert x[n:] == [-1] * (len(x) - n), x
        out.append(x[:n])
    B, H, T, _ = blocks.shape
    return [[out[(b * H + h) * T:(b * H + h + 1) * T] for h in range(H)] for b in range(B)]


@pytest.mark.parametrize("D,G,T,top,first,recent", [(64, 1, 1, 4, 1, 1), (128, 6, 1, 7, 1, 2), (256, 6, 3, 16, 0, 0), (64, 20, 2, 3, 2, 0),
                                                    (128, 2, 40, 5, 1, 1), (256, 3, 1, 64, 1, 1), (64, 2, 70, 1, 0, 0),
                                                    (64, 100, 1, 6, 1, 1), (128, 48, 3, 5, 0, 1), (64, 16, 5, 9, 1, 1),
                                                    (64, 2, 230, 3, 1, 1), (256, 3, 215, 5, 0, 1), (128, 17, 110, 4, 1, 0)])
def test_select_and_attend(dev, D, G, T, top, first, recent):
    gen = torch.Generator().manual_seed(D + 7 * G + T + top)
    H = 2
    lens = [max(n, T) for n in (2000, 1, 64, 1281, 700)]
    B = len(lens)
    k, v = keys(gen, B, H, max(lens), D)
    c = fill(dev, k, v, lens)
    q = rand(gen, B, H * G, T, D)
    blocks = tsa.kv8_select(q.to(dev), c, ints(lens, dev), top, first=first, recent=recent)
    lists = chosen(q, k, lens, [T] * B, top, first, recent)
    assert as_lists(blocks) == lists
    o = tsa.attn_kv8_blocks_fwd(q.to(dev), c, ints(lens, dev), blocks)
    want, tol = expect(q, k, v, lens, [T] * B, True, lists=lists)
    check_out(o.cpu(), want, tol, "sparse")


def test_select_ties_and_odd_blocks(dev):
    """Equal blocks (the lowest index first), a block with a NaN, one without a page, a group of zeros
    or with an infinity, padding, and a max_len that is too short."""
    gen = torch.Generator().manual_seed(31)
    D, L = 64, 64 * 30 + 3
    k, v = keys(gen, 1, 1, L, D)
    for i in (3, 9, 12, 20, 28):
        k[0, 0, 64 * i:64 * i + 64] = k[0, 0, :64]
    k[0, 0, 64 * 5 + 7, 3] = math.nan
    c = fill(dev, k, v, [L])
    c.table[0, 9] = -1
    pages = [i != 9 for i in range(31)]
    T = 4
    q = rand(gen, 1, 2, T, D)
    q[0, :, 1] = 0
    q[0, 0, 2, 0] = math.inf
    for top in (2, 5, 28, 29, 30, 31, 40):
        got = tsa.kv8_select(q.to(dev), c, ints([L], dev), top, first=1, recent=0)
        assert as_lists(got) == chosen(q, k, [L], [T], top, 1, 0, pages=pages), top
    got = tsa.kv8_select(q.to(dev), c, ints([L], dev), 9, first=0, recent=1, max_len=64 * 11)
    assert as_lists(got) == chosen(q, k, [L], [T], 9, 0, 1, pages=pages, scored=11)
    kept = torch.full((1, 1, T, 6), 77, dtype=torch.int32, device=dev)
    tsa.kv8_select(q.to(dev), c, ints([L], dev), 6, ints([2], dev), out=kept)
    assert bool((kept[:, :, 2:] == 77).all())
    assert as_lists(kept[:, :, :2]) == chosen(q[:, :, :2], k, [L], [2], 6, 1, 1, pages=pages)
    # in front of the sequence there is no block
    got = tsa.kv8_select(q.to(dev), c, ints([2], dev), 6)
    assert as_lists(got)[0][0] == [[], [], [0], [0]]


def test_listed_blocks_of_the_callers(dev):
    """Lists in any order, with repeats, numbers that are no block, blocks behind the query, and none."""
    gen = torch.Generator().manual_seed(32)
    D, G, T, L = 128, 3, 5, 64 * 7 + 30
    k, v = keys(gen, 1, 1, L, D)
    c = fill(dev, k, v, [L])
    q = rand(gen, 1, G, T, D)
    lists = [[[[3, 0, 7, 1], [2, 2, 7, 7], [-1, 1 << 30, 5, -(1 << 31)], [-1] * 4, [8, 9, 6, 400]]]]
    o = tsa.attn_kv8_blocks_fwd(q.to(dev), c, ints([L], dev), ints(lists, dev))
    want, tol = expect(q, k, v, [L], [T], True, lists=lists)
    check_out(o.cpu(), want, tol, "listed")
    assert not bool(o[0, :, 3].any())


@pytest.mark.parametrize("nb,top", [(500, 40), (1999, 300), (3001, 40), (9000, 1), (9000, 8500)])
def test_select_many_blocks(dev, nb, top):
    """More blocks than one workgroup scores at once or holds in registers, against the definition in
    whole numbers."""
    gen = torch.Generator().manual_seed(33)
    D, G = 64, 4
    L = 64 * nb + 9
    c = tsa.Kv8Cache(1, 1, D, L, device=dev)
    c.k_sum.copy_(torch.randint(-127, 128, c.k_sum.shape, generator=gen, dtype=torch.int8))
    c.k_sum_scale.copy_(torch.rand(c.k_sum_scale.shape, generator=gen) + 0.5)
    c.k_sum[100:1500:7] = c.k_sum[99]  # many equals
    c.k_sum_scale[100:1500:7] = c.k_sum_scale[99]
    q = rand(gen, 1, G, 2, D)
    first, recent = (2, 3) if top > 5 else (0, 0)
    got = tsa.kv8_select(q.to(dev), c, ints([L], dev), top, first=first, recent=recent).cpu()
    m, s = c.k_sum.cpu().double()[:, 0], c.k_sum_scale.cpu().numpy()[:, 0]
    for t in range(2):
        x = q[0, :, t].double()
        score = (torch.round(127 * x / x.abs().max()) @ m.T).amax(0).numpy().astype(np.float32) * s
        own = nb
        rank = [(np.inf if i < first or i >= own - recent else score[i], -i) for i in range(own + 1)]
        assert got[0, 0, t].tolist() == sorted(-r[1] for r in sorted(rank, reverse=True)[:top])


# ---------------------------------------------------------------------------------------
# together, as a server uses them
# ---------------------------------------------------------------------------------------
def test_serving_run(dev):
    """Two prompts of unequal length, then tokens one at a time, dense and over selected blocks, the
    whole step captured once and replayed with the program's own work between: every replay equals
    the eager call bit for bit, and the eager ones the definition."""
    gen = torch.Generator().manual_seed(41)
    D, H, G, B, steps = 128, 2, 3, 2, 6
    prompt, cap = [190, 61], 512
    k, v = keys(gen, B, H, cap, D)
    qp, qs = rand(gen, B, H * G, 190, D), rand(gen, steps, B, H * G, 1, D)
    gs = rand(gen, steps, B, H * G, 1, D)

    def start():
        c = tsa.Kv8Cache(B, H, D, cap, device=dev)
        n = ints(prompt, dev)
        tsa.kv8_write(c, k[:, :, :190].to(dev), v[:, :, :190].to(dev), n, n)
        return c, n

    def step(c, st):
        st["len"].add_(1)
        tsa.kv8_write(c, st["k"], st["v"], st["len"])
        tsa.attn_kv8_fwd(st["q"], c, st["len"], gate=st["gate"], out=st["dense"], ws=st["ws"])
        tsa.kv8_select(st["q"], c, st["len"], 3, out=st["blocks"], ws=st["ws"])
        tsa.attn_kv8_blocks_fwd(st["q"], c, st["len"], st["blocks"], gate=st["gate"], out=st["sparse"], ws=st["ws"])

    def feed(st, i):
        at = [n + i for n in prompt]
        st["k"].copy_(torch.stack([k[b, :, at[b]:at[b] + 1] for b in range(B)]))
        st["v"].copy_(torch.stack([v[b, :, at[b]:at[b] + 1] for b in range(B)]))
        st["q"].copy_(qs[i])
        st["gate"].copy_(gs[i])

    def state(c, n):
        z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
        ws = max(tsa.kv8_workspace_bytes(c, 1, H * G), tsa.kv8_workspace_bytes(c, 1, H * G, top=3))
        return {"len": n, "k": z(B, H, 1, D), "v": z(B, H, 1, D), "q": z(B, H * G, 1, D), "gate": z(B, H * G, 1, D),
                "dense": z(B, H * G, 1, D), "sparse": z(B, H * G, 1, D),
                "blocks": torch.zeros(B, H, 1, 3, dtype=torch.int32, device=dev),
                "ws": torch.empty(max(ws, 1), dtype=torch.uint8, device=dev)}

    c, n = start()
    o = tsa.attn_kv8_fwd(qp.to(dev), c, n, n)
    want, tol = expect(qp, k, v, prompt, prompt, True)
    for b in range(B):
        check_out(o[b, :, :prompt[b]].cpu(), want[b, :, :prompt[b]], tol[b, :, :prompt[b]], ("prompt", b))
        assert not bool(o[b, :, prompt[b]:].any())
    eager, st = [], state(c, n.clone())
    for i in range(steps):
        feed(st, i)
        step(c, st)
        lens = [p + i + 1 for p in prompt]
        eager.append({x: st[x].clone() for x in ("dense", "blocks", "sparse")})
        want, tol = expect(qs[i], k, v, lens, [1] * B, True, gs[i])
        check_out(st["dense"].cpu(), want, tol, ("dense", i))
        lists = chosen(qs[i], k, lens, [1] * B, 3, 1, 1)
        assert as_lists(st["blocks"]) == lists
        want, tol = expect(qs[i], k, v, lens, [1] * B, True, gs[i], lists=lists)
        check_out(st["sparse"].cpu(), want, tol, ("sparse", i))

    c, n = start()
    st = state(c, n.clone())
    feed(st, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a warm-up before the capture, taken back afterwards
        step(c, st)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c, st)
    c2, n2 = start()
    st["len"].copy_(n2)
    for name in ("k", "v", "k_scale", "v_scale", "k_sum", "k_sum_scale", "k_open", "v_open"):
        getattr(c, name).copy_(getattr(c2, name))
    for i in range(steps):
        feed(st, i)
        graph.replay()
        torch.cuda.synchronize()
        for x in eager[i]:
            assert torch.equal(st[x], eager[i][x]), (x, i)
        (qp.to(dev).float().sum() + 1).item()


def test_another_stream(dev):
    """Calls on a stream of their own, workspaces made by the binding."""
    gen = torch.Generator().manual_seed(42)
    D, L = 64, 3000
    k, v = keys(gen, 1, 1, L, D)
    q = rand(gen, 1, 4, 1, D)
    s = torch.cuda.Stream()
    args = [x.to(dev) for x in (k, v, q)]
    n = ints([L], dev)
    c = tsa.Kv8Cache(1, 1, D, L, device=dev)
    s.wait_stream(torch.cuda.current_stream())
    tsa.kv8_write(c, args[0], args[1], n, stream=s)
    blocks = torch.zeros(1, 1, 1, 8, dtype=torch.int32, device=dev)
    s.wait_stream(torch.cuda.current_stream())
    tsa.kv8_select(args[2], c, n, 8, out=blocks, stream=s)
    o, oq = torch.zeros_like(args[2]), torch.zeros_like(args[2])
    s.wait_stream(torch.cuda.current_stream())
    tsa.attn_kv8_fwd(args[2], c, n, out=o, stream=s)
    tsa.attn_kv8_blocks_fwd(args[2], c, n, blocks, out=oq, stream=s)
    own = tsa.attn_kv8_fwd(args[2], c, n, stream=s)
    s.synchronize()
    assert torch.equal(own, o)
    want, tol = expect(q, k, v, [L], [1], True)
    check_out(o.cpu(), want, tol, "dense")
    lists = chosen(q, k, [L], [1], 8, 1, 1)
    assert as_lists(blocks) == lists
    want, tol = expect(q, k, v, [L], [1], True, lists=lists)
    check_out(oq.cpu(), want, tol, "sparse")


def test_refused_tensors(dev):
    c = tsa.Kv8Cache(2, 2, 64, 128, device=dev)
    z = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    n, x, q = ints([1, 1], dev), z(2, 2, 1, 64), z(2, 4, 1, 64)
    for bad in (z(2, 2, 1, 64, t=torch.float32), z(2, 3, 1, 64), z(1, 2, 1, 64), z(2, 2, 1, 128), x.cpu(),
                z(2, 2, 1, 128)[..., ::2]):
        with pytest.raises(ValueError):
            tsa.kv8_write(c, bad, x, n)
        with pytest.raises(ValueError):
            tsa.kv8_write(c, x, bad, n)
    for bad in (ints([1], dev), n.long(), n.cpu(), ints([1, 1, 1, 1], dev)[::2]):
        with pytest.raises(ValueError):
            tsa.kv8_write(c, x, x, bad)
        with pytest.raises(ValueError):
            tsa.attn_kv8_fwd(q, c, n, bad)
    with pytest.raises(TypeError):
        tsa.kv8_write(c, x, x, None)
    odd = z(2 * 2 * 64 + 8)[1:1 + 256].view(2, 2, 1, 64)  # rows that are not 16-byte aligned
    with pytest.raises(tsa.TsaError) as e:
        tsa.kv8_write(c, odd, x, n)
    assert e.value.code == tsa.TSA_ERR_ARG
    with pytest.raises(tsa.TsaError) as e:
        tsa.attn_kv8_fwd(z(2, 3, 1, 64), c, n)
    assert e.value.code == tsa.TSA_ERR_SHAPE
    with pytest.raises(ValueError):
        tsa.attn_kv8_fwd(q, c, n, out=z(2, 4, 2, 64))
    with pytest.raises(tsa.TsaError) as e:  # an output broadcast over heads
        tsa.attn_kv8_fwd(q, c, n, out=z(2, 1, 1, 64).expand(2, 4, 1, 64))
    assert e.value.code == tsa.TSA_ERR_ARG
    with pytest.raises(ValueError):
        tsa.attn_kv8_blocks_fwd(q, c, n, ints([0], dev).view(1, 1, 1, 1))
    with pytest.raises(ValueError):
        tsa.attn_kv8_blocks_fwd(q, c, n, z(2, 2, 1, 3, t=torch.int64))
    with pytest.raises(tsa.TsaError) as e:
        tsa.kv8_select(q, c, n, 2, first=1, recent=1)
    assert e.value.code == tsa.TSA_ERR_ARG
    need = tsa.kv8_workspace_bytes(c, 1, 4, top=8)
    with pytest.raises(tsa.TsaError) as e:
        tsa.kv8_select(q, c, n, 8, ws=z(need - 1, t=torch.uint8))
    assert e.value.code == tsa.TSA_ERR_WORKSPACE
