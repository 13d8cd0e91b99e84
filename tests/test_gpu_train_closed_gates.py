"""The backward pass where the gate makes gradients small: dO = sigmoid(gate) d_out has fp16's full precision in every
row, and d is made of the same dO as dP."""
import math

import pytest
import torch

import train_oracle as orc
import tsa
from test_gpu_attn_train import make, within

pytestmark = pytest.mark.gpu


def bounds(do, q, k, v, o, lse, gate, causal):
    """The oracle's gradients, and bounds of their errors that do not grow with the call's largest row:
      dO  rounded once, below fp16's normal range to half of 2^-24 times the row's power of two: 2^-32 of the row's norm (at
          least 2^7 as it is kept), or 2^-25 where the norm is above that; sigmoid within 2^-18
      P   rounded; half a step of 2^-24 under a factor of 2^15, less the row's power above the largest row's: 2^-40 times
          twice the ratio of the norms, at least once
      dS  rounded from the rounded P; half a step of 2^-24 at the bound's power of two (2^13 of it at least): 2^-38"""
    Hkv, Tk, D = k.shape[1:]
    G, Tq, c = q.shape[1] // Hkv, q.shape[2], 1 / math.sqrt(k.shape[3])
    want, _ = orc.backward(do, q, k, v, o, lse, gate, causal=causal)
    q, do, o, lse, sig = q.double(), do.double(), o.double(), lse.double()[..., None], torch.sigmoid(gate.double())
    k, v = orc.heads(k, G), orc.heads(v, G)
    see = orc.visible(q.shape[0], Tq, Tk, None, None, causal, q.device)
    g, d = do * sig, (do * o).sum(-1, keepdim=True)
    p = torch.where(see, torch.exp(c * (q @ k.transpose(2, 3)) - lse), 0.0)
    dp = torch.where(see, g @ v.transpose(2, 3), 0.0)
    ds = p * (dp - d)
    norm = g.norm(dim=-1, keepdim=True)
    eg = (orc.U + 2.0 ** -18) * g.abs() + torch.where(norm < 2.0 ** 7, 2.0 ** -32 * norm, 2.0 ** -25)
    rel = torch.expm1(2 * ((D + 4) * 2.0 ** -23 * c * (q.abs() @ k.abs().transpose(2, 3)) + 2.0 ** -22 * (lse.abs() + 64)))
    floor_p = 2.0 ** -40 * torch.where(norm > 0, (2 * norm.amax() / norm).clamp_min(1), 1.0)
    ep = torch.where(see, p * (orc.U + rel) + floor_p, 0.0)
    # (d is made of the rounded dO: the row's sum of dS stays 0, and the rounding of dO is that of dP - d)
    edp = eg @ v.abs().transpose(2, 3) + torch.where(sig > 0, eg * (o / sig).abs(), 0.0).sum(-1, keepdim=True) + \
        (D + 8) * 2.0 ** -23 * (g.abs() @ v.abs().transpose(2, 3) + (do * o).abs().sum(-1, keepdim=True))
    most = float(norm.amax() * v.norm(dim=-1).amax() + d.abs().amax())
    eds = torch.where(see, ds.abs() * (2 * orc.U + rel) + (p + ep) * edp + floor_p * (dp - d).abs() + most * 2.0 ** -38, 0.0)
    group = lambda x: x.view(x.shape[0], Hkv, G, *x.shape[2:]).sum(2)  # noqa: E731
    n = (max(Tq * G, Tk) + 8) * 2.0 ** -23
    bv = group(ep.transpose(2, 3) @ g.abs() + (p + ep).transpose(2, 3) @ eg + n * (p.transpose(2, 3) @ g.abs()))
    bq = c * (eds @ k.abs() + n * (ds.abs() @ k.abs()))
    bk = c * group(eds.transpose(2, 3) @ q.abs() + n * (ds.abs().transpose(2, 3) @ q.abs()))
    return [(name, want[name], 1.01 * b + orc.U * (want[name].abs() + b) + 2.0 ** -25) for name, b in (("dq", bq), ("dk", bk), ("dv", bv))]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("closed", [0.0, -6.0, -9.0])
def test_small_gradients_behind_a_gate(dev, D, closed):
    """d_out near 2^-14, the same in all queries, and one gate for all: dO is some steps of 2^-24, and each column's
    rounding would go into dV as it is."""
    q, k, v, gate, do = make(dev, 90, 1, 2, 1, 2048, 64, D, True, size=0.5)
    do = (2.0 ** -14 * (1 + 0.3 * do[:, :, :1]).clamp(0.2, 2)).expand_as(do).contiguous()
    gate, v = torch.full_like(gate, closed), v * 64
    o, lse = tsa.attn_train_fwd(q, k, v, gate, causal=False)
    grads = tsa.attn_bwd(do, q, k, v, o, lse, gate, causal=False)
    for (name, want, bound), got in zip(bounds(do, q, k, v, o, lse, gate, False), grads):
        within(name, got, want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Tq,Tk,causal", [(600, 600, True), (1300, 4000, True), (333, 100, False)])
def test_rows_of_all_sizes(dev, D, Tq, Tk, causal):
    """Queries whose gradients lie up to 2^16 apart, in one call."""
    q, k, v, gate, do = make(dev, 91, 1, 4, 1, Tq, Tk, D, True, size=0.7)
    gen = torch.Generator(device=dev)
    gen.manual_seed(92)
    do = (do.float() * 2.0 ** (-16 * torch.rand(1, 4, Tq, 1, generator=gen, device=dev))).half()
    o, lse = tsa.attn_train_fwd(q, k, v, gate, causal=causal)
    grads = tsa.attn_bwd(do, q, k, v, o, lse, gate, causal=causal)
    for (name, want, bound), got in zip(bounds(do, q, k, v, o, lse, gate, causal), grads):
        within(name, got, want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_two_sizes_of_one_gradient(dev, D):
    """d_out and d_out 2^7, each within its bounds.  (Not the same bits: a row's power of two is added to its statistic, whose
    rounding, 2^-24 of their sum, then differs, and a P now and then with it.)"""
    q, k, v, gate, do = make(dev, 93, 1, 2, 1, 2048, 64, D, True, size=0.5)
    gate, less = gate - 3, do.clamp(-7, 7) * 2.0 ** -7
    o, lse = tsa.attn_train_fwd(q, k, v, gate, causal=False)
    for x in (less, less * 2.0 ** 7):
        grads = tsa.attn_bwd(x, q, k, v, o, lse, gate, causal=False)
        for (name, want, bound), got in zip(bounds(x, q, k, v, o, lse, gate, False), grads):
            within(name, got, want, bound)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_single_key_behind_a_closed_gate(dev, D):
    """One key: dS is what o's rounding leaves, sum d_out (sigma v - o).  Off by dO's rounding of that, 2^-11 of sum |d_out|
    |sigma v - o|; the sums in 32 bits (D / 8 products a lane, 3 steps; 16 products of an instruction, D / 16 of those) and
    sigma of a gate of -15 (2^-24 times 15 log2(e), twice), 40 2^-24 in all, of sum |dO| |v|; dS's and the result's own rounding."""
    q, k, v, gate, do = make(dev, 94, 500, 4, 4, 1, 1, D, True)
    q, k, do, gate = q * 2.0 ** -10, k * 2000, do * 0.05, torch.full_like(gate, -15.0)
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    dq = tsa.attn_bwd(do, q, k, v, o, lse, gate)[0]
    x, y, w, sig, c = do.double(), o.double(), v.double(), torch.sigmoid(gate.double()), D ** -0.5
    ds = (x * sig * w).sum(-1, keepdim=True) - (x * y).sum(-1, keepdim=True)
    off = 2.0 ** -11 * (x * (y - sig * w)).abs().sum(-1, keepdim=True) + \
        (D / 8 + 3 + 16 + D / 16 + 40) * 2.0 ** -24 * (x * sig * w).abs().sum(-1, keepdim=True) + 2.0 ** -11 * ds.abs()
    want = c * ds * k.double()
    assert ((dq.double() - want).abs() <= 1.01 * c * off * k.double().abs() + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()
    assert want.abs().mean() > 2.0 ** -22  # (what is looked at is there)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_gates_at_the_ends(dev, D):
    """Gates that close or open fully, and whole rows of them: sigmoid is 0 or 1, and nothing becomes NaN."""
    q, k, v, gate, do = make(dev, 95, 1, 2, 1, 70, 70, D, True)
    ends = [-65504.0, -300.0, -88.7, -80.0, -30.0, 30.0, 80.0, 88.7, 65504.0, float("inf"), -float("inf")]
    gate[..., :len(ends)] = torch.tensor(ends, device=dev).half()
    for i, x in enumerate(ends):
        gate[:, :, 3 * i] = x
    o, lse = tsa.attn_train_fwd(q, k, v, gate)
    grads = tsa.attn_bwd(do, q, k, v, o, lse, gate)
    for (name, want, bound), got in zip(bounds(do, q, k, v, o, lse, gate.double().clamp(-1e3, 1e3), True), grads):
        within(name, got, want, bound)
    want = do.double() * o.double() * (1 - torch.sigmoid(gate.double()))
    assert ((grads[3].double() - want).abs() <= 1.01 * orc.U * want.abs() + 2.0 ** -20 * want.abs() + 2.0 ** -25).all()
    shut = torch.isin(torch.arange(70, device=dev), torch.tensor([3 * i for i, x in enumerate(ends) if x <= -300], device=dev))
    assert not grads[0][:, :, shut].any()
