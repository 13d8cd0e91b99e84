"""Rotary positions (tsa_rope) against 64-bit oracles."""
import math

import pytest
import torch

import train_oracle as orc
import tsa

pytestmark = pytest.mark.gpu


def rows(dev, seed, B, H, T, D, dtype=torch.float16, layout="bhsd"):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    shape = (B, H, T, D) if layout == "bhsd" else (B, T, H, D)
    x = torch.randn(*shape, generator=gen, device=dev).to(dtype)
    return x if layout == "bhsd" else x.transpose(1, 2)


def check(rope, f, amp, x, got, pos, n=None, back=False):
    want = orc.rotate(x, pos, f, amp, rope.interleaved, back)
    bound = orc.rotate_bound(x, want, pos, f, abs(amp), rope.interleaved)
    off = (got.double() - want).abs()
    if n is not None:
        pad = (torch.arange(x.shape[2], device=x.device) >= n.long()[:, None])[:, None, :, None].expand_as(x)
        assert not got[pad].any()
        off = torch.where(pad, 0.0, off)
    assert (off <= bound).all(), float((off / bound.clamp_min(1e-30)).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (64, 20), (64, 2), (128, 128), (128, 32), (128, 30), (128, 126), (256, 64), (256, 256), (256, 96)])
def test_forward_and_gradient(dev, D, rot, interleaved, dtype):
    q, k = rows(dev, 1, 2, 5, 37, D, dtype), rows(dev, 2, 2, 3, 37, D, dtype, "bshd")
    rope = tsa.Rope(D, rot=rot, interleaved=interleaved)
    f, amp = orc.freqs(rot)
    pos = torch.arange(37, device=dev).expand(2, 37)
    for back, fn in ((False, tsa.rope_fwd), (True, tsa.rope_bwd)):
        for x, y in zip((q, k), fn(rope, q, k)):
            check(rope, f, amp, x, y, pos, back=back)
            assert torch.equal(x[..., rot:], y[..., rot:])
        a, b = q.clone(), k.clone()
        assert fn(rope, a, b, q_out=a, k_out=b)[0] is a
        for x, y in zip(fn(rope, q, k), (a, b)):  # in place: the same bits
            assert torch.equal(x, y)
        assert torch.equal(fn(rope, q)[0], a) and fn(rope, q)[1] is None


SCALED = [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0), dict(scaling="yarn", factor=16.0, orig_len=4096),
          dict(scaling="wavelength", factor=8.0, orig_len=8192, low=1.0, high=4.0),
          dict(scaling="yarn", factor=1.0, orig_len=100), dict(scaling="yarn", factor=3.0, orig_len=1, beta_fast=4.0, beta_slow=0.5)]


@pytest.mark.parametrize("kw", SCALED, ids=lambda k: f"{k['scaling']}-{k['factor']:g}-{k.get('orig_len', 0)}")
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (256, 64)])
def test_scaled(dev, D, rot, kw):
    rope = tsa.Rope(D, rot=rot, base=5e5, **kw)
    f, amp = orc.freqs(rot, base=5e5, **kw)
    assert abs(rope.amp - amp) <= 2.0 ** -24 * amp
    got = torch.tensor(rope.turns, dtype=torch.float64) * 2 * math.pi
    # the oracle's powers are off by some 2^-51; the table by half of 2^-64 turns
    assert ((got - f).abs() <= 2.0 ** -49 * f + 2.0 ** -60).all()
    x = rows(dev, 3, 1, 4, 65, D)
    pos = torch.arange(65, dtype=torch.int32, device=dev)[None] * 2003
    check(rope, got, rope.amp, x, tsa.rope_fwd(rope, x, pos=pos)[0], pos)


def test_far_positions(dev):
    """Angles of positions up to both ends of 32 bits keep their precision (the oracle in exact whole
    numbers: a table entry times a position, mod 2^64)."""
    D = 128
    rope = tsa.Rope(D, base=1e6)
    table = [int(round(t * 2.0 ** 64)) for t in rope.turns]
    table = [x & ((1 << 64) - 1) for x in rope.freq.tolist()]
    where = [0, 1, -1, 131071, 131072, 1000003, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, -12345]
    pos = torch.tensor([where], dtype=torch.int32, device=dev)
    x = rows(dev, 4, 1, 3, len(where), D, torch.float32)
    got = tsa.rope_fwd(rope, x, pos=pos)[0].double().cpu()
    turns = torch.tensor([[((p * f) % (1 << 64)) / 2.0 ** 64 for f in table] for p in where], dtype=torch.float64)
    c, s = torch.cos(2 * math.pi * turns), torch.sin(2 * math.pi * turns)
    a, b = x.double().cpu()[..., :64], x.double().cpu()[..., 64:]
    want = torch.cat([a * c - b * s, b * c + a * s], -1)
    assert ((got - want).abs() <= 2.0 ** -21 * (a.abs() + b.abs()).repeat(1, 1, 1, 2)).all()


def test_positions(dev):
    """Positions of rows: given, from the cache's counts, or the row's number; padding."""
    D, B, T = 128, 4, 6
    q, k = rows(dev, 5, B, 4, T, D, layout="bshd"), rows(dev, 6, B, 2, T, D)
    rope, (f, amp) = tsa.Rope(D, rot=64, interleaved=True), orc.freqs(64)
    t = torch.arange(T, device=dev)
    ln = torch.tensor([6, 4097, 131072, 3], dtype=torch.int32, device=dev)
    n = torch.tensor([6, 1, 0, 9], dtype=torch.int32, device=dev)  # 9 is taken as T
    taken = n.clamp(0, T)
    for kw, pos, pad in ((dict(len=ln), (ln - T)[:, None] + t, None), (dict(len=ln, n_new=n), (ln - taken)[:, None] + t, taken),
                         (dict(n_new=n), t.expand(B, T), taken), (dict(pos=(ln[:, None] * 3 - t).int().contiguous(), n_new=n), ln[:, None] * 3 - t, taken)):
        for x, y in zip((q, k), tsa.rope_fwd(rope, q, k, **kw)):
            check(rope, f, amp, x, y, pos, pad)
    out = torch.full_like(q, 5.0)
    tsa.rope_fwd(rope, q, n_new=n, q_out=out)
    for b in range(B):
        assert (out[b, :, int(taken[b]):] == 5).all()


def test_padding_is_not_read(dev):
    x = rows(dev, 7, 2, 2, 8, 64)
    n = torch.tensor([3, 8], dtype=torch.int32, device=dev)
    y = x.clone()
    y[0, :, 3:] = math.nan
    rope = tsa.Rope(64)
    a, b = tsa.rope_fwd(rope, x, n_new=n)[0], tsa.rope_fwd(rope, y, n_new=n)[0]
    assert torch.equal(a, b) and torch.isfinite(a).all()


def test_strides_and_streams(dev):
    rope = tsa.Rope(128, rot=96)
    with pytest.raises(tsa.TsaError) as e:  # rows that begin off 16 bytes are refused
        tsa.rope_fwd(rope, torch.randn(5, 3, 7, 300, device=dev).half()[..., 16:144].permute(1, 2, 0, 3))
    assert e.value.code == tsa.TSA_ERR_ARG
    big = torch.randn(5, 3, 7, 304, device=dev).half()
    x = big[..., 16:144].permute(1, 2, 0, 3)  # [3, 7, 5, 128]
    want = tsa.rope_fwd(rope, x.contiguous())[0]
    assert torch.equal(tsa.rope_fwd(rope, x)[0], want)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = tsa.rope_fwd(rope, x, stream=s)[0]
    s.synchronize()
    assert torch.equal(got, want)
    one = x[:, :1].expand(3, 7, 5, 128)
    assert torch.equal(tsa.rope_fwd(rope, one)[0], tsa.rope_fwd(rope, one.contiguous())[0])


def test_there_and_back(dev):
    """The gradient's rotation undoes the rotation up to two roundings of each."""
    x = rows(dev, 8, 1, 3, 50, 256, torch.float32)
    for interleaved in (False, True):
        rope = tsa.Rope(256, interleaved=interleaved)
        y = tsa.rope_bwd(rope, tsa.rope_fwd(rope, x)[0])[0]
        assert (y - x).abs().max() <= 2.0 ** -20 * x.abs().max()


def test_step_into_the_cache(dev):
    """A server's step: rotated queries and keys, the key written to the 8-bit cache, attention over it;
    captured, and replayed as the sequences grow."""
    B, Hq, Hkv, D = 3, 4, 2, 128
    rope = tsa.Rope(D, rot=64, base=1e6)
    cache = tsa.Kv8Cache(B, Hkv, D, 256)
    n = torch.tensor([5, 70, 1], dtype=torch.int32, device=dev)
    q, k, v = rows(dev, 9, B, Hq, 1, D), rows(dev, 10, B, Hkv, 1, D), rows(dev, 11, B, Hkv, 1, D)
    past_k, past_v = rows(dev, 12, B, Hkv, 80, D), rows(dev, 13, B, Hkv, 80, D)
    tsa.kv8_write(cache, tsa.rope_fwd(rope, past_k, n_new=n)[0], past_v, n, n)
    ws = torch.empty(max(1, tsa.kv8_workspace_bytes(cache, 1, Hq)), dtype=torch.uint8, device=dev)
    qr, kr, o = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
    ln = n.clone()

    def run():
        tsa.rope_fwd(rope, q, k, len=ln, q_out=qr, k_out=kr)
        tsa.kv8_write(cache, kr, v, ln)
        tsa.attn_kv8_fwd(qr, cache, ln, out=o, ws=ws)

    ln += 1
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    f, amp = orc.freqs(64, base=1e6)
    for i in range(4):
        q.copy_(rows(dev, 30 + i, B, Hq, 1, D))
        ln += 1
        g.replay()
        torch.cuda.synchronize()
        check(rope, f, amp, q, qr, (ln - 1)[:, None])
        check(rope, f, amp, k, kr, (ln - 1)[:, None])
        keys, values = tsa.kv8_read(cache, ln)
        for b in range(B):
            m = int(ln[b])
            s = (qr[b, :, 0].double().view(Hkv, Hq // Hkv, D) @ keys[b, :, :m].double().transpose(1, 2)) / math.sqrt(D)
            want = torch.softmax(s, -1) @ values[b, :, :m].double()
            # P, the codes' values and o rounded to fp16: 2^-11 each of sum P |v| (at most max |v|), and scores 2^-11 of theirs
            tol = 4 * 2.0 ** -11 * float(values[b, :, :m].abs().max()) * (1 + float(s.abs().max()))
            assert (o[b, :, 0].double().view(Hkv, Hq // Hkv, D) - want).abs().max() <= tol
