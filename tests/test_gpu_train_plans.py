"""The training pair's ways of dealing out work that small calls do not take: key tiles whose queries go over several
workgroups, with lengths, in workspaces of exactly their size and in one that two graphs share; whole query tiles of
padded batches."""
import math

import pytest
import torch

import train_oracle as orc
import tsa
from test_gpu_attn_train import lens, make, step, within
from test_gpu_train_edges import outputs, pair, same

pytestmark = pytest.mark.gpu

SPLIT = [  # Hq, Hkv, Tq, Tk, lengths of queries and keys
    (8, 2, 600, 600, [600, 1, 333], [600, 47, 590]),
    (8, 2, 600, 600, [0, 600, 333], [600, 600, 100]),
    (4, 1, 1100, 1100, [1100, 700, 33], [1100, 700, 33]),
    (6, 2, 800, 333, [800, 31, 64], [333, 333, 1]),
    (6, 1, 500, 2000, [500, 77, 500], [2000, 1999, 0]),
]


def splits(B, Hq, Hkv, Tq, Tk, D, causal):
    """Whether a key tile's queries are split: two parts of dK and dV at least are in the workspace."""
    return tsa.attn_bwd_workspace_bytes(B, Hq, Hkv, Tq, Tk, D, gated=False, causal=causal) >= 2 * 2 * 4 * B * Hkv * Tk * D


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", SPLIT, ids=lambda c: "-".join(str(x) for x in c[:4]) + f"-{c[4][0]}")
def test_split_key_tiles_with_lengths(dev, D, causal, case):
    Hq, Hkv, Tq, Tk, lq, lk = case
    assert splits(3, Hq, Hkv, Tq, Tk, D, causal)
    q, k, v, gate, do = make(dev, 110, 3, Hq, Hkv, Tq, Tk, D, True, "bshd")
    lq, lk = lens(dev, lq), lens(dev, lk)
    o, lse, grads = step(q, k, v, gate, do, lq=lq, lk=lk, causal=causal)
    # no padding is read: the same with NaN there
    for x, n in ((q, lq), (gate, lq), (do, lq), (k, lk), (v, lk), (o, lq)):
        x.masked_fill_((torch.arange(x.shape[2], device=dev) >= n.long()[:, None])[:, None, :, None], math.nan)
    for a, b in zip(grads, tsa.attn_bwd(do, q, k, v, o, lse, gate, len_q=lq, len_k=lk, causal=causal)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("padded", [True, False])
def test_workspace_with_parts(dev, D, gate, padded):
    size = (2, 6, 1, 500, 700, D)
    assert splits(*size, True)
    q, k, v, gate, do = make(dev, 111, *size, gate)
    n = lens(dev, [500, 321]) if padded else None
    m = lens(dev, [700, 400]) if padded else None
    o, lse = tsa.attn_train_fwd(q, k, v, gate, len_q=n, len_k=m)
    bytes_ = tsa.attn_bwd_workspace_bytes(*size, gated=gate is not None)
    want = tsa.attn_bwd(do, q, k, v, o, lse, gate, len_q=n, len_k=m)
    for fill in (0, 255):
        ws = torch.full((bytes_ + 4096,), fill, dtype=torch.uint8, device=dev)
        ws[bytes_:] = 77
        got = tsa.attn_bwd(do, q, k, v, o, lse, gate, len_q=n, len_k=m, ws=ws[:bytes_])
        assert (ws[bytes_:] == 77).all()
        assert same(got, want)
    oracle, bound = orc.backward(do, q, k, v, o, lse, gate, len_q=n, len_k=m)
    for name, got, rows in zip(("dq", "dk", "dv", "dg"), want, (n, m, m, n)):
        if got is not None:
            within(name, got, oracle[name], bound[name], rows)


def test_two_graphs_share_a_workspace_with_parts(dev):
    shapes = [(2, 8, 2, 600, 600, 128, True), (1, 6, 1, 800, 333, 256, False)]
    assert all(splits(*s[:6], True) for s in shapes)
    ins = [make(dev, 112 + i, *s) for i, s in enumerate(shapes)]
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
            for a, b in zip(x, make(dev, 120 + 2 * i + j, *shapes[j])):
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


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (7, 7)])
def test_whole_tiles_of_a_padded_batch(dev, D, causal, Hq, Hkv):
    """More query tiles than any split takes, with lengths (B Hq a multiple of 8, spread over the XCDs, and not)."""
    B, T = (8, 1500) if Hq == 8 else (9, 1500)
    q, k, v, gate, _ = make(dev, 113, B, Hq, Hkv, T, T, D, True, "bshd")
    n = lens(dev, [1500, 1, 700, 1499, 0, 65, 1100, 333, 1500][:B])
    o, lse = tsa.attn_train_fwd(q, k, v, gate, len_q=n, len_k=n, causal=causal)
    for b in range(B):  # (a sequence at a time: the oracle's scores are of all heads and rows)
        rows = [x[b:b + 1] for x in (q, k, v, gate)]
        want, want_l, bo, bl = orc.forward(*rows, len_q=n[b:b + 1], len_k=n[b:b + 1], causal=causal)
        within("o", o[b:b + 1], want, bo, n[b:b + 1])
        m = int(n[b])
        assert ((lse[b:b + 1].double() - want_l).abs() <= bl + 2.0 ** -22 * want_l.abs())[:, :, :m].all() and not lse[b, :, m:].any()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_captured_step_of_a_padded_batch(dev, D):
    """Rotary positions, forward, backward and back in one graph, with split key tiles, replayed with other lengths."""
    B, Hq, Hkv, T = 3, 8, 2, 600
    assert splits(B, Hq, Hkv, T, T, D, True)
    x = make(dev, 130, B, Hq, Hkv, T, T, D, True, "bshd")
    q, k, v, gate, do = x
    n = lens(dev, [600, 1, 333])
    rope = tsa.Rope(D, rot=32)
    ws = torch.empty(tsa.attn_bwd_workspace_bytes(B, Hq, Hkv, T, T, D, gated=True), dtype=torch.uint8, device=dev)
    new = lambda: [torch.zeros_like(q), torch.zeros_like(k), *outputs(x)]  # noqa: E731

    def run(y, ws):
        qr, kr, o, lse, dq, dk, dv, dg = y
        tsa.rope_fwd(rope, q, k, n_new=n, q_out=qr, k_out=kr)
        tsa.attn_train_fwd(qr, kr, v, gate, len_q=n, len_k=n, out=o, lse=lse)
        tsa.attn_bwd(do, qr, kr, v, o, lse, gate, len_q=n, len_k=n, dq=dq, dk=dk, dv=dv, dgate=dg, ws=ws)
        tsa.rope_bwd(rope, dq, dk, n_new=n, q_out=dq, k_out=dk)

    got = new()
    run(got, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(got, ws)
    for i, length in enumerate(([600, 1, 333], [0, 600, 599], [77, 600, 600], [600, 0, 64])):
        n.copy_(lens(dev, length))
        for a, b in zip(x, make(dev, 131 + i, B, Hq, Hkv, T, T, D, True, "bshd")):
            a.copy_(b)
        for a in got:
            a.zero_()
        g.replay()
        torch.cuda.synchronize()
        want = new()
        run(want, None)
        assert same(got, want) and any(a.any() for a in got)
