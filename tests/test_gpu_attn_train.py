"""Attention's training pair (tsa_attn_train_fwd, tsa_attn_bwd) against 64-bit oracles: gradients of
queries, keys, values and gate, padded batches, strides, lengths from one, rows that see no key."""
import math

import pytest
import torch

import train_oracle as orc
import tsa

pytestmark = pytest.mark.gpu


def make(dev, seed, B, Hq, Hkv, Tq, Tk, D, gate, layout="bhsd", size=1.0, grad=1.0):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def rows(H, T, f):
        shape = (B, H, T, D) if layout == "bhsd" else (B, T, H, D)
        x = (f * torch.randn(*shape, generator=gen, device=dev)).half()
        return x if layout == "bhsd" else x.transpose(1, 2)

    return rows(Hq, Tq, size), rows(Hkv, Tk, size), rows(Hkv, Tk, 1.0), rows(Hq, Tq, 1.0) if gate else None, rows(Hq, Tq, grad)


def lens(dev, x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


def within(name, got, want, bound, rows=None):
    """got is within bound of want; rows behind `rows` are 0."""
    off = (got.double() - want).abs()
    if rows is not None:
        pad = torch.arange(got.shape[2], device=got.device) >= rows.long()[:, None]
        pad = pad.view(pad.shape[0], 1, pad.shape[1], *[1] * (got.dim() - 3)).expand_as(got)
        assert not got[pad].any(), f"{name}: padding was written"
        off = torch.where(pad, 0.0, off)
    assert torch.isfinite(got).all(), name
    worst = (off / bound).max()
    assert worst <= 1, f"{name}: off by {float(worst):.2f} bounds, {float(off.max()):.3g}"


def step(q, k, v, gate, do, lq=None, lk=None, causal=True, scale=None):
    """Forward and backward, each against its oracle."""
    kw = dict(len_q=lq, len_k=lk, causal=causal, scale=scale)
    o, lse = tsa.attn_train_fwd(q, k, v, gate, **kw)
    want_o, want_l, bo, bl = orc.forward(q, k, v, gate, **kw)
    within("o", o, want_o, bo, lq)
    empty = torch.isinf(want_l)
    pad = torch.zeros_like(empty) if lq is None else (torch.arange(q.shape[2], device=q.device) >= lq.long()[:, None])[:, None].expand_as(empty)
    assert (lse[empty & ~pad] == -math.inf).all() and not lse[pad].any()
    seen = ~empty & ~pad
    assert ((lse.double() - want_l).abs() <= bl + 2.0 ** -22 * want_l.abs())[seen].all()
    grads = tsa.attn_bwd(do, q, k, v, o, lse, gate, **kw)
    want, bound = orc.backward(do, q, k, v, o, lse, gate, **kw)
    for name, got, n in zip(("dq", "dk", "dv", "dg"), grads, (lq, lk, lk, lq)):
        if got is not None:
            within(name, got, want[name], bound[name], n)
    return o, lse, grads


SIZES = [  # B, Hq, Hkv, Tq, Tk, D, gate, causal, layout
    (1, 1, 1, 1, 1, 64, False, True, "bhsd"),
    (2, 2, 1, 1, 77, 128, True, True, "bhsd"),
    (1, 3, 3, 2, 2, 256, False, False, "bhsd"),
    (1, 2, 2, 31, 31, 64, False, True, "bhsd"),
    (1, 2, 2, 32, 32, 128, False, True, "bshd"),
    (1, 2, 1, 33, 33, 256, True, True, "bshd"),
    (2, 4, 2, 64, 64, 64, False, False, "bhsd"),
    (1, 2, 2, 65, 130, 128, False, True, "bhsd"),
    (1, 2, 2, 127, 129, 256, False, True, "bhsd"),
    (1, 4, 1, 128, 128, 64, True, True, "bshd"),
    (1, 4, 1, 200, 200, 128, True, True, "bshd"),
    (1, 6, 1, 150, 150, 256, True, True, "bhsd"),
    (1, 2, 2, 257, 255, 64, False, False, "bhsd"),
    (3, 3, 1, 300, 700, 128, False, True, "bshd"),
    (1, 2, 1, 513, 513, 256, False, True, "bhsd"),
    (2, 5, 5, 401, 401, 64, False, True, "bshd"),
    (1, 12, 4, 640, 640, 64, True, True, "bhsd"),
    (1, 1, 1, 1025, 1025, 128, False, False, "bhsd"),
    (1, 8, 1, 1, 4099, 64, False, True, "bhsd"),
    (1, 1, 1, 2000, 3, 128, False, False, "bhsd"),
    (8, 8, 8, 300, 300, 64, False, True, "bshd"),  # more key tiles than a split takes
]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(str(x) for x in s))
def test_step(dev, size):
    B, Hq, Hkv, Tq, Tk, D, gate, causal, layout = size
    q, k, v, gate, do = make(dev, 1, B, Hq, Hkv, Tq, Tk, D, gate, layout)
    step(q, k, v, gate, do, causal=causal)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_padded_batch(dev, D, causal):
    """Lengths from 0, fewer keys than queries (rows that see no key), NaN and infinities in padding."""
    lq, lk = [70, 0, 1, 33, 64, 5, 70], [90, 90, 0, 7, 64, 65, 1]
    q, k, v, gate, do = make(dev, 2, 7, 4, 2, 70, 90, D, True, "bshd")
    lq, lk = lens(dev, lq), lens(dev, lk)
    q_pad = (torch.arange(70, device=dev) >= lq.long()[:, None])[:, None, :, None]
    k_pad = (torch.arange(90, device=dev) >= lk.long()[:, None])[:, None, :, None]
    for x, pad in ((q, q_pad), (gate, q_pad), (do, q_pad), (k, k_pad), (v, k_pad)):
        x.masked_fill_(pad, math.nan)
        x[:, :, 1::2].masked_fill_(pad[:, :, 1::2], math.inf)
    clean = [torch.where(pad, 0, x) for x, pad in ((q, q_pad), (k, k_pad), (v, k_pad), (gate, q_pad), (do, q_pad))]
    o, lse, grads = step(*[c.transpose(1, 2).contiguous().transpose(1, 2) for c in clean], lq=lq, lk=lk, causal=causal)
    o2, lse2 = tsa.attn_train_fwd(q, k, v, gate, len_q=lq, len_k=lk, causal=causal)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    dirty_o, dirty_l = o2.clone(), lse2.clone()
    dirty_o.masked_fill_(q_pad, math.nan)
    dirty_l.masked_fill_(q_pad[..., 0].expand_as(dirty_l), math.nan)
    for a, b in zip(grads, tsa.attn_bwd(do, q, k, v, dirty_o, dirty_l, gate, len_q=lq, len_k=lk, causal=causal)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_padding_is_left_as_it_was(dev, D):
    q, k, v, gate, do = make(dev, 3, 2, 2, 1, 40, 50, D, True)
    lq, lk = lens(dev, [7, 33]), lens(dev, [9, 50])
    o, lse = torch.full_like(q, 3.0), torch.full(q.shape[:3], 5.0, device=dev)
    tsa.attn_train_fwd(q, k, v, gate, len_q=lq, len_k=lk, out=o, lse=lse)
    out = [torch.full_like(x, 7.0) for x in (q, k, v, gate)]
    tsa.attn_bwd(do, q, k, v, o, lse, gate, len_q=lq, len_k=lk, dq=out[0], dk=out[1], dv=out[2], dgate=out[3])
    for b in range(2):
        assert (o[b, :, int(lq[b]):] == 3).all() and (lse[b, :, int(lq[b]):] == 5).all()
        for x, n in zip(out, (lq, lk, lk, lq)):
            assert (x[b, :, int(n[b]):] == 7).all()
    o2, lse2 = tsa.attn_train_fwd(q, k, v, gate, len_q=lq, len_k=lk)
    for x, y in zip(out, tsa.attn_bwd(do, q, k, v, o2, lse2, gate, len_q=lq, len_k=lk)):
        assert torch.equal(torch.where(x == 7.0, 0.0, x), torch.where(y == 7.0, 0.0, y))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("grad", [2.0 ** -17, 1e-3, 300.0])
def test_gradients_of_any_size(dev, D, grad):
    """fp16's range: the gradients' precision does not fall with their size."""
    q, k, v, gate, do = make(dev, 4, 1, 2, 1, 500, 500, D, False, size=0.5, grad=grad)
    step(q, k, v, gate, do)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_sharp_and_large(dev, D):
    """Probabilities near 0 and 1: large scores, outliers in keys and values."""
    q, k, v, gate, do = make(dev, 5, 1, 4, 2, 190, 190, D, False, size=3.0)
    v[:, :, ::17] *= 40
    step(q, k, v, gate, do)
    step(q, k, v, gate, do, scale=2.0 / math.sqrt(D), causal=False)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_strides(dev, D):
    """Rows out of larger tensors, heads of one tensor side by side, a key head shared by stride 0."""
    B, Hq, Hkv, T = 2, 4, 2, 100
    gen = torch.Generator(device=dev)
    gen.manual_seed(6)
    packed = torch.randn(T, B, Hq + 2 * Hkv + Hq, D + 16, generator=gen, device=dev).half()
    view = packed[..., 8:8 + D].permute(1, 2, 0, 3)
    q, k, v, gate = view[:, :Hq], view[:, Hq:Hq + Hkv], view[:, Hq + Hkv:Hq + 2 * Hkv], view[:, Hq + 2 * Hkv:]
    do = torch.randn(B, Hq, T, D, generator=gen, device=dev).half()
    dense = [x.contiguous() for x in (q, k, v, gate)]
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    o2, lse2 = tsa.attn_train_fwd(*dense)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    whole = torch.zeros(T, B, 2 * Hq + 2 * Hkv, D, dtype=torch.float16, device=dev).permute(1, 2, 0, 3)
    outs = dict(dq=whole[:, :Hq], dk=whole[:, Hq:Hq + Hkv], dv=whole[:, Hq + Hkv:Hq + 2 * Hkv], dgate=whole[:, Hq + 2 * Hkv:])
    tsa.attn_bwd(do, q, k, v, o, lse, gate, **outs)
    for a, b in zip(outs.values(), tsa.attn_bwd(do, *dense[:3], o2, lse2, dense[3])):
        assert torch.equal(a, b)
    one = dense[1][:, :1]
    shared = one.expand(B, Hkv, T, D)
    a = tsa.attn_bwd(do, dense[0], shared, dense[2], *tsa.attn_train_fwd(dense[0], shared, dense[2]))
    b = tsa.attn_bwd(do, dense[0], shared.contiguous(), dense[2], *tsa.attn_train_fwd(dense[0], shared.contiguous(), dense[2]))
    for x, y in zip(a[:3], b[:3]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_same_as_the_plain_forward(dev, D, causal):
    """The training form and tsa_attn_gqa_fwd run the same products; the sums differ by their rounding."""
    q, k, v, gate, _ = make(dev, 7, 1, 4, 2, 700, 700, D, True)
    o, _ = tsa.attn_train_fwd(q, k, v, gate, causal=causal)
    plain = tsa.attn_gqa_fwd(q, k, v, gate, causal=causal)
    want, _, bound, _ = orc.forward(q, k, v, gate, causal=causal)
    assert ((o.double() - plain.double()).abs() <= 2 * bound).all()


def test_gradient_against_differences(dev):
    """d/dx sum(w o) by central differences of the 64-bit forward."""
    q, k, v, gate, do = make(dev, 8, 1, 2, 1, 20, 23, 64, True)
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    grads = tsa.attn_bwd(do, q, k, v, o, lse, gate)
    _, bound = orc.backward(do, q, k, v, o, lse, gate)
    xs = [q.double(), k.double(), v.double(), gate.double()]
    loss = lambda *x: (do.double() * orc.forward(*x)[0]).sum()  # noqa: E731
    h = 1e-4
    gen = torch.Generator().manual_seed(9)
    for i, name in enumerate(("dq", "dk", "dv", "dg")):
        for _ in range(10):
            at = tuple(int(torch.randint(n, (1,), generator=gen)) for n in xs[i].shape)
            ends = []
            for sign in (1, -1):
                moved = [x.clone() for x in xs]
                moved[i][at] += sign * h
                ends.append(loss(*moved))
            slope = (ends[0] - ends[1]) / (2 * h)
            # o is rounded to fp16: d_i and dgate take that on (2^-11 of |do| |o| a row); differences are off by h^2
            rounding = 2.0 ** -11 * float((do.double() * o.double()).abs().sum(-1).max()) * 3
            assert abs(float(grads[i][at]) - float(slope)) <= float(bound[name][at]) + rounding + 1e-6, (name, at)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_same_bits_again_and_on_another_stream(dev, D):
    q, k, v, gate, do = make(dev, 10, 2, 6, 2, 333, 444, D, True, "bshd")
    first = tsa.attn_train_fwd(q, k, v, gate)
    grads = tsa.attn_bwd(do, q, k, v, *first, gate)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    again = tsa.attn_train_fwd(q, k, v, gate, stream=s)
    more = tsa.attn_bwd(do, q, k, v, *again, gate, stream=s)
    s.synchronize()
    for a, b in zip((*first, *grads), (*again, *more)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_workspace_is_enough_and_holds_nothing_over(dev, D):
    q, k, v, gate, do = make(dev, 11, 1, 6, 2, 150, 333, D, True)
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    n = tsa.attn_bwd_workspace_bytes(1, 6, 2, 150, 333, D, gated=True)
    want = tsa.attn_bwd(do, q, k, v, o, lse, gate)
    for fill in (0, 255):
        ws = torch.full((n + 4096,), fill, dtype=torch.uint8, device=dev)
        ws[n:] = 77
        got = tsa.attn_bwd(do, q, k, v, o, lse, gate, ws=ws[:n])
        assert (ws[n:] == 77).all()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    with pytest.raises(tsa.TsaError) as e:
        tsa.attn_bwd(do, q, k, v, o, lse, gate, ws=ws[:n - 16])
    assert e.value.code == tsa.TSA_ERR_WORKSPACE


def test_captured_step(dev):
    """Forward and backward in one graph, replayed with new inputs between eager calls."""
    q, k, v, gate, do = make(dev, 12, 2, 4, 2, 130, 130, 128, True)
    ws = torch.empty(tsa.attn_bwd_workspace_bytes(2, 4, 2, 130, 130, 128, gated=True), dtype=torch.uint8, device=dev)
    o, lse = torch.empty_like(q), torch.empty(q.shape[:3], device=dev)
    outs = [torch.empty_like(x) for x in (q, k, v, gate)]

    def run():
        tsa.attn_train_fwd(q, k, v, gate, out=o, lse=lse)
        tsa.attn_bwd(do, q, k, v, o, lse, gate, dq=outs[0], dk=outs[1], dv=outs[2], dgate=outs[3], ws=ws)

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for i in range(4):
        for x, y in zip((q, k, v, gate, do), make(dev, 20 + i, 2, 4, 2, 130, 130, 128, True)):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (o, lse, *outs)]
        first = tsa.attn_train_fwd(q, k, v, gate)
        for a, b in zip(got, (*first, *tsa.attn_bwd(do, q, k, v, *first, gate))):
            assert torch.equal(a, b)


def test_whole_layer(dev):
    """Rotary positions, forward, backward and back through the rotation, as a layer's step runs them."""
    B, Hq, Hkv, T, D = 2, 6, 2, 150, 128
    q, k, v, gate, do = make(dev, 13, B, Hq, Hkv, T, T, D, True, "bshd")
    n = lens(dev, [150, 99])
    rope = tsa.Rope(D, rot=64)
    qr, kr = tsa.rope_fwd(rope, q, k, n_new=n)
    o, lse = tsa.attn_train_fwd(qr, kr, v, gate, len_q=n, len_k=n)
    dq, dk, dv, dg = tsa.attn_bwd(do, qr, kr, v, o, lse, gate, len_q=n, len_k=n)
    xq, xk = tsa.rope_bwd(rope, dq, dk, n_new=n)
    # the same from the 64-bit oracles, each on what the step before left in fp16
    want, bound = orc.backward(do, qr, kr, v, o, lse, gate, len_q=n, len_k=n)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv), ("dg", dg)):
        within(name, got, want[name], bound[name], n)
    f, amp = orc.freqs(64)
    pos = torch.arange(T, device=dev).expand(B, T)
    for got, x in ((xq, dq), (xk, dk)):
        y = orc.rotate(x, pos, f, amp, False, back=True)
        within("rotated back", got, y, orc.rotate_bound(x, y, pos, f, amp, False) + 2.0 ** -25, n)


NO_NUMBERS = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Tq,Tk,at", [(200, 200, 100), (150, 187, 186), (70, 70, 33), (513, 513, 480), (90, 40, 20), (1100, 1100, 1000)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_no_numbers_in_a_hidden_key(dev, D, Tq, Tk, at, where):
    """A token's infinity or NaN reaches the queries that see it, and no others: not o, lse or dq of queries
    in front of it, which the mask hides it from."""
    q, k, v, gate, do = make(dev, 14, 1, 2, 1, Tq, Tk, D, True)
    want_o, want_l, bo, bl = orc.forward(q, k, v, gate)
    clean = tsa.attn_train_fwd(q, k, v, gate)
    want, bound = orc.backward(do, q, k, v, *clean, gate)
    x = {"k": k, "v": v}[where]
    for i, bad in enumerate(NO_NUMBERS):
        kept = x[:, :, at].clone()
        x[:, :, at, (5 + 7 * i) % D] = bad
        o, lse = tsa.attn_train_fwd(q, k, v, gate)
        dq = tsa.attn_bwd(do, q, k, v, o, lse, gate)[0]
        x[:, :, at] = kept
        before = max(0, at - (Tk - Tq))  # queries in front of the token
        rows = slice(0, before)
        assert ((o.double() - want_o).abs() <= bo)[:, :, rows].all()
        seen = torch.isfinite(want_l[:, :, rows])
        assert ((lse.double() - want_l).abs()[:, :, rows] <= (bl + 2.0 ** -22 * want_l.abs())[:, :, rows])[seen].all()
        # (o of these rows may differ in its last bit from the clean call's, and d with it: twice the bound, and that of d)
        slack = 2.0 ** -10 * (do.double() * clean[0].double()).abs().sum(-1, keepdim=True) * k.double().abs().amax() / math.sqrt(D)
        assert ((dq.double() - want["dq"]).abs() <= 2 * bound["dq"] + slack)[:, :, rows].all()
        # what sees it: an infinite key's score is minus infinity where the query has the other sign there, a
        # weight of 0, so only the others' rows hold no number
        hit = torch.ones(1, 2, Tq, dtype=torch.bool, device=dev)
        if where == "k" and not math.isnan(bad):
            hit = q[..., (5 + 7 * i) % D].double() * bad > 0
        hit[:, :, rows] = False
        assert (~torch.isfinite(o)).any(-1)[hit].all()
        assert (~torch.isfinite(dq)).any(-1)[hit].all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Tq,Tk,at", [(200, 200, 100), (150, 187, 3), (70, 70, 33), (513, 513, 500), (90, 40, 70), (1100, 1100, 40)])
@pytest.mark.parametrize("where", ["q", "do"])
def test_no_numbers_in_a_query(dev, D, Tq, Tk, at, where):
    """A query's (or its gradient's) infinity or NaN reaches the keys that it sees, and no others."""
    q, k, v, gate, do = make(dev, 15, 1, 2, 1, Tq, Tk, D, False)
    clean = tsa.attn_train_fwd(q, k, v)
    want, bound = orc.backward(do, q, k, v, *clean)
    # without the row at all: what keys in front of it get from the others is not looked at
    x = {"q": q, "do": do}[where]
    for i, bad in enumerate(NO_NUMBERS):
        kept = x[:, :, at].clone()
        x[:, :, at, (3 + 11 * i) % D] = bad
        o, lse = tsa.attn_train_fwd(q, k, v)
        dq, dk, dv, _ = tsa.attn_bwd(do, q, k, v, o, lse)
        x[:, :, at] = kept
        first = max(0, at + (Tk - Tq) + 1)  # the first key that the query does not see
        for name, got in (("dk", dk), ("dv", dv)):
            assert ((got.double() - want[name]).abs() <= bound[name])[:, :, first:].all(), name
            assert first == 0 or (~torch.isfinite(got[:, :, :first])).any(-1).all(), name
        others = torch.arange(Tq, device=dev) != at
        assert ((dq.double() - want["dq"]).abs() <= bound["dq"])[:, :, others].all()
        assert (~torch.isfinite(dq[:, :, at])).any() or first == 0
