"""The training forward where one key outweighs all others, a long sequence's first one for instance: the small weights
keep their bits."""
import math

import pytest
import torch

import train_oracle as orc
import tsa
from test_gpu_attn_train import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Tq,Tk,causal", [(40, 60000, True), (300, 60000, True), (2100, 5000, False), (40, 777, True), (1500, 1500, True)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_key_above_all_others(dev, D, Tq, Tk, causal):
    """The first key's score lies 13.83 (2^-24 times 16.5) and 17 above the others', which are equal, and its value is 0: o is
    what the small weights make, each rounded alike.  A weight is rounded by 2^-11 of itself or half a step of 2^-24; it
    is kept times 2^7, and the row's sum is at least that of the largest, 2^7 (the maximum that the exponentials are taken
    against may lie below it, never above), so the step counts 2^-32.  The rest as in the oracle's bound."""
    q, k, v, _, _ = make(dev, 100, 1, 2, 1, Tq, Tk, D, False)
    v = v.abs() * 4
    q[..., 0] = 4
    k.zero_()
    v[:, :, 0] = 0
    for above in (13.83, 17.0):
        k[:, :, 0, 0] = above * math.sqrt(D) / 4
        o, lse = tsa.attn_train_fwd(q, k, v, causal=causal)
        want, want_l, _, bl = orc.forward(q, k, v, causal=causal)
        s = q.double() @ orc.heads(k, 2).transpose(2, 3) / math.sqrt(D)
        p = torch.where(orc.visible(1, Tq, Tk, None, None, causal, dev), torch.exp(s - want_l[..., None]), 0.0)
        mag = p @ orc.heads(v, 2)
        worst = (D + 4) * 2.0 ** -23 * above + 2.0 ** -22 * want_l.abs()[..., None]
        bound = orc.U * (mag + want.abs()) + (2 * torch.expm1(2 * worst) + (Tk + 8) * 2.0 ** -23) * mag + 2.0 ** -32 * v.double().sum(2, keepdim=True) + 2.0 ** -25
        assert ((o.double() - want).abs() <= bound).all(), float(((o.double() - want).abs() / bound).max())
        assert ((lse.double() - want_l).abs() <= bl + 2.0 ** -22 * want_l.abs()).all()
