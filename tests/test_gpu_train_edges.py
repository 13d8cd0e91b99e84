"""The training pair and rotary positions where callers share, stretch or overflow things: a workspace of
two graphs, two streams at once, lengths out of range, offsets past 32 bits, many sequences, infinities
among the last values."""
import math

import pytest
import torch

import train_oracle as orc
import tsa
from test_gpu_attn_train import lens, make, step

pytestmark = pytest.mark.gpu


def pair(x, outs, ws, **kw):
    q, k, v, gate, do = x
    o, lse, dq, dk, dv, dg = outs
    tsa.attn_train_fwd(q, k, v, gate, out=o, lse=lse, **kw)
    tsa.attn_bwd(do, q, k, v, o, lse, gate, dq=dq, dk=dk, dv=dv, dgate=dg, ws=ws, **kw)


def outputs(x):
    q, k, v, gate, _ = x
    return [torch.zeros_like(q), torch.zeros(q.shape[:3], device=q.device)] + [None if y is None else torch.zeros_like(y) for y in (q, k, v, gate)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b) if x is not None)


def test_two_graphs_share_a_workspace(dev):
    shapes = [(1, 4, 2, 200, 200, 128, True), (2, 6, 1, 90, 333, 128, False)]
    ins = [make(dev, 30 + i, *s) for i, s in enumerate(shapes)]
    ws = torch.empty(max(tsa.attn_bwd_workspace_bytes(*s[:6], gated=s[6]) for s in shapes), dtype=torch.uint8, device=dev)
    outs, graphs = [outputs(x) for x in ins], []
    for x, y in zip(ins, outs):
        pair(x, y, ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pair(x, y, ws)
        graphs.append(g)
    for i in range(3):
        for j, x in enumerate(ins):
            for a, b in zip(x, make(dev, 40 + 2 * i + j, *shapes[j])):
                if a is not None:
                    a.copy_(b)
        for y in outs:
            for a in y:
                if a is not None:
                    a.fill_(math.nan)
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for x, y in zip(ins, outs):
            want = outputs(x)
            pair(x, want, None)
            assert same(y, want)


def test_two_streams_at_once(dev):
    ins = [make(dev, 50 + i, 1, 4, 2, 700, 700, 64 * (i + 1), True, "bshd") for i in range(2)]
    want, got = [outputs(x) for x in ins], [outputs(x) for x in ins]
    for x, y in zip(ins, want):
        pair(x, y, None)
    wss = [torch.empty(tsa.attn_bwd_workspace_bytes(1, 4, 2, 700, 700, x[0].shape[3], gated=True), dtype=torch.uint8, device=dev) for x in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    for _ in range(4):
        for x, y, w, s in zip(ins, got, wss, streams):
            pair(x, y, w, stream=s)
    torch.cuda.synchronize()
    assert same(got[0], want[0]) and same(got[1], want[1])


@pytest.mark.parametrize("causal", [True, False])
def test_lengths_out_of_range(dev, causal):
    """A length below 0 is 0, one past the rows all of them."""
    x = make(dev, 60, 3, 2, 2, 100, 150, 64, True)
    a, b = outputs(x), outputs(x)
    pair(x, a, None, len_q=lens(dev, [-5, 1000, 70]), len_k=lens(dev, [40, 2 ** 31 - 1, -2 ** 31]), causal=causal)
    pair(x, b, None, len_q=lens(dev, [0, 100, 70]), len_k=lens(dev, [40, 150, 0]), causal=causal)
    assert same(a, b) and not a[0][0].any() and not a[0][2, :, :70].any()


@pytest.mark.parametrize("stride_b,stride_t", [(256, 2 ** 24), (2 ** 32 + 8192, 8192)])
def test_offsets_past_32_bits(dev, stride_b, stride_t):
    B, Hq, Hkv, T, D = 2, 2, 1, 140, 64
    big = torch.zeros(stride_b + (T - 1) * stride_t + 8192, dtype=torch.half, device=dev)
    x = make(dev, 61, B, Hq, Hkv, T, T, D, True)
    place = iter(range(0, 8192, 512))

    def far(y):
        z = big.as_strided(y.shape, (stride_b, D, stride_t, 1), next(place))
        z.copy_(y)
        return z

    want, far_x = outputs(x), [far(y) for y in x]
    got = [y if y.dtype == torch.float32 else far(y) for y in outputs(x)]
    pair(x, want, None)
    pair(far_x, got, None)
    assert same(got, want)
    for rot in (64, 20):
        rope = tsa.Rope(D, rot=rot, interleaved=rot == 20)
        assert same(tsa.rope_fwd(rope, far_x[0], far_x[1]), tsa.rope_fwd(rope, x[0], x[1]))


@pytest.mark.parametrize("D", [64, 256])
def test_many_sequences(dev, D):
    step(*make(dev, 62, 70000, 1, 1, 1, 1, D, False))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,Tq,Tk", [(1, 200, 200), (1, 30, 77), (2, 1100, 1100), (1, 2100, 2100)])
@pytest.mark.parametrize("causal", [True, False])
def test_infinite_values(dev, D, B, Tq, Tk, causal):
    """Infinities of one column of many tokens' values, the last one's among them: what sees one has an infinity
    there, and what does not, and every other column, has its number."""
    q, k, v, gate, _ = make(dev, 63, B, 2, 1, Tq, Tk, D, False)
    col = D // 2 + 3
    at = torch.arange(Tk - 1, -1, -97, device=dev)
    kept = v[:, :, at, col].clone()
    v[:, :, at, col] = math.inf
    o, lse = tsa.attn_train_fwd(q, k, v, causal=causal)
    v[:, :, at, col] = 0.0
    want, want_l, bound, bl = orc.forward(q, k, v, causal=causal)
    sees = orc.visible(B, Tq, Tk, None, None, causal, dev)[..., at].any(-1).expand(B, 2, Tq)
    assert (o[..., col][sees] == math.inf).all()
    off = (o.double() - want).abs() <= bound
    off[..., col] |= sees
    assert off.all()
    assert ((lse.double() - want_l).abs() <= bl + 2.0 ** -22 * want_l.abs()).all()
    v[:, :, at, col] = kept
