"""The backward pass of gradients of any size: P keeps its bits however large they are."""
import math

import pytest
import torch

import train_oracle as orc
import tsa
from test_gpu_attn_train import make, within

pytestmark = pytest.mark.gpu

SIZES = [  # Hq, Hkv, Tq, Tk, D, causal, values' size
    (2, 1, 200, 4096, 64, False, 1.0),
    (2, 1, 200, 4096, 128, False, 1.0),
    (2, 1, 200, 4096, 256, False, 1.0),
    (2, 2, 2100, 2100, 64, True, 1.0),
    (4, 1, 1300, 4000, 128, True, 1.0),  # key tiles in parts
    (4, 1, 1300, 4000, 256, True, 1.0),
    (1, 1, 250, 65536, 128, False, 32.0),
    (1, 1, 250, 65536, 256, False, 32.0),
]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "-".join(str(x) for x in s))
def test_gradients_grow_with_their_input(dev, size):
    """d_out times a power of two is every gradient times it: each step of the call scales exactly (P does not change, and
    dS's power of two goes with the bound), except where the smaller gradient is at most 2^-14: below that it
    is rounded to 2^-24 (up to 2^-14 itself, too), half a step off, and the larger one by 2^-11 of itself.
    At D <= 128 dQ's P has dS's power of two in its exponential's argument, whose rounding (2^-24 of some tens)
    moves a dS to its neighbour now and then: there both are held to their bounds."""
    Hq, Hkv, Tq, Tk, D, causal, big = size
    q, k, v, _, do = make(dev, 80, 1, Hq, Hkv, Tq, Tk, D, False, size=0.5)
    v, do = v * big, do.clamp(-7, 7)
    o, lse = tsa.attn_train_fwd(q, k, v, causal=causal)
    for by in (-4, 5, 10, 13):
        # (from the smaller one up: fp16 holds do 2^-4 rounded where that is below 2^-14, but every x 2^by of an x it holds)
        less = do * 2.0 ** min(by, 0)
        by = abs(by)
        base, more = (tsa.attn_bwd(x, q, k, v, o, lse, causal=causal) for x in (less, less * 2.0 ** by))
        for name, x, y in zip(("dq", "dk", "dv"), base, more):
            if name == "dq" and D <= 128:
                continue
            x, y = x.double() * 2.0 ** by, y.double()
            small = (x.abs() <= 2.0 ** (by - 14)) | (y.abs() <= 2.0 ** -14)
            assert torch.equal(x[~small], y[~small]), (name, by)
            assert ((x - y).abs() <= 1.01 * (2.0 ** (by - 25) + 2.0 ** -25) + orc.U * y.abs())[small].all(), (name, by)
        if D <= 128:
            for x, dq in ((less, base[0]), (less * 2.0 ** by, more[0])):
                want, bound = orc.backward(x, q, k, v, o, lse, causal=causal)
                within("dq", dq, want["dq"], bound["dq"])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_keys(dev, D):
    """The smallest of these calls against 64 bits."""
    q, k, v, _, do = make(dev, 81, 1, 2, 1, 200, 4096, D, False, size=0.5)
    o, lse = tsa.attn_train_fwd(q, k, v, causal=False)
    want, bound = orc.backward(do, q, k, v, o, lse, causal=False)
    for name, got in zip(("dq", "dk", "dv"), tsa.attn_bwd(do, q, k, v, o, lse, causal=False)):
        within(name, got, want[name], bound[name])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_row_far_larger_than_the_others(dev, D):
    """One query's gradient 2^12 times as large: the values that it does not see get what they got without it, to
    the last bit (P is the same).  dS has its steps from the largest row's bound: 2^-39 of it (half a step of 2^-24 at
    2^14) for each query, and dP - d the same 32-bit sums."""
    T, at = 2050, 3
    q, k, v, _, do = make(dev, 82, 1, 2, 1, T, T, D, False, size=0.5)
    o, lse = tsa.attn_train_fwd(q, k, v)
    first = tsa.attn_bwd(do, q, k, v, o, lse)
    want, bound = orc.backward(do, q, k, v, o, lse)
    do[:, :, at] *= 4096
    dq, dk, dv, _ = tsa.attn_bwd(do, q, k, v, o, lse)
    assert torch.equal(dv[:, :, at + 1:], first[2][:, :, at + 1:])
    most = do.double().norm(dim=-1).amax() * v.double().norm(dim=-1).amax() + (do.double() * o.double()).sum(-1).abs().amax()
    c, step = 1 / math.sqrt(D), float(most) * 2.0 ** -38
    more = c * step * q.double().abs().sum((1, 2), keepdim=True)  # (both query heads, all queries)
    assert ((dk.double() - want["dk"]).abs() <= bound["dk"] + more)[:, :, at + 1:].all()
    rows = torch.arange(T, device=dev) != at
    more = c * step * k.double().abs().sum(2, keepdim=True)
    assert ((dq.double() - want["dq"]).abs() <= bound["dq"] + more)[:, :, rows].all()
