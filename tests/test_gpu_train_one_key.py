"""Where a query sees a single key, dS is what rounding o to fp16 leaves: the forward's o has to be the
rounding of its value, not of a neighbour's."""
import pytest
import torch

import tsa
from test_gpu_attn_train import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rounding_of_a_gated_value(dev, D):
    """o = sigmoid(gate) v in 32 bits is off by less than 3 2^-24 of it on average (sigmoid at most 2.4, 0.6 on
    average; the one exponential, 2^x of the rounding of a score below 8, at most 2.8; three roundings of at most 1), so
    it falls to the other side of a rounding in fewer than 3 2^-24 / 2^-12 of the elements, each of them a
    value within 8 2^-24 of the middle between two fp16 numbers."""
    q, k, v, gate, _ = make(dev, 70, 500, 4, 4, 1, 1, D, True)
    gate *= 3
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    exact = torch.sigmoid(gate.double()) * v.double()
    want = exact.half()
    other = o != want
    assert other.double().mean() < 3 * 2.0 ** -24 / 2.0 ** -12
    middle = (o.double() + want.double()) / 2
    assert ((exact - middle).abs() <= 4 * 2.0 ** -23 * exact.abs() + 2.0 ** -45)[other].all()


def test_gates_at_the_ends(dev):
    """Gates of any size, infinities and NaN among them."""
    q, k, v, gate, _ = make(dev, 71, 2, 2, 2, 8, 8, 64, True)
    ends = [-65504.0, -300.0, -80.0, -17.0, 0.0, 17.0, 80.0, 65504.0, float("inf"), -float("inf")]
    gate[..., :10] = torch.tensor(ends, device=dev).half()
    gate[..., 10] = float("nan")
    o, _ = tsa.attn_train_fwd(q, k, v, gate)
    plain, _ = tsa.attn_train_fwd(q, k, v)
    want = torch.sigmoid(gate.double()) * plain.double()  # (plain is rounded once already)
    assert torch.isnan(o[..., 10]).all()
    o, want, plain = (torch.cat([x[..., :10], x[..., 11:]], -1) for x in (o, want, plain))
    assert ((o.double() - want).abs() <= 1.01 * 2.0 ** -10 * want.abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_gradient_of_a_single_key(dev, D):
    """dS = dO.v - d is what o's rounding leaves, 2^-12 of either.  Off by: dO's rounding of that (2^-11 of
    sum |do| |o - sigma v|), the sums in 32 bits (d: D / 8 products a lane, 3 steps; dP: 16 products of an
    instruction, D / 16 of those; each 2^-24 of sum |dO| |v|, and 8 2^-24 for 1 / sigma), and dS's and dq's own rounding to fp16."""
    q, k, v, gate, do = make(dev, 72, 500, 4, 4, 1, 1, D, True)
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    dq, dk, _, _ = tsa.attn_bwd(do, q, k, v, o, lse, gate)
    g, x, y, w = (t.double() for t in (gate, do, o, v))
    sig, c = torch.sigmoid(g), D ** -0.5
    ds = (x * sig * w).sum(-1, keepdim=True) - (x * y).sum(-1, keepdim=True)
    off = 2.0 ** -11 * (x * (y - sig * w)).abs().sum(-1, keepdim=True) + \
        (D / 8 + 3 + 16 + D / 16 + 8) * 2.0 ** -24 * (x * sig * w).abs().sum(-1, keepdim=True) + 2.0 ** -11 * ds.abs()
    for got, other in ((dq, k), (dk, q)):
        want = c * ds * other.double()
        assert ((got.double() - want).abs() <= c * off * other.double().abs() + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()
