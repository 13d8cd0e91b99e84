"""Attention's training pair and rotary positions in 64 bits from their definitions, and what the
kernels' roundings can make of them.

Bounds (u = 2^-11, half a step of fp16; every sum in fp32 is taken as off by its length times 2^-23
of the sum of magnitudes):
  scores      es = (D + 4) 2^-23 c |q|.|k| + 2^-22 |lse|: so P is off by the factor e^(2 es) - 1 at most
  o           P rounded to fp16: u sum P|v|; es; P below fp16's normal range 2^-24 each; o rounded: u |o|
  dO          with a gate rounded once: u |dO| + 2^-25
  dV          P rounded, dO rounded, es, P's floor f = max(2^-40, bound 2^-38) (half of fp16's least step
              times the power of two that the bound of |dS| allows), dV rounded
  dS          P rounded, dS rounded, es, dP's own sum and dO's rounding, d's sum, the floor bound 2^-38
"""
import math

import torch

U = 2.0 ** -11


def heads(x, G):
    return x.double().repeat_interleave(G, 1)


def visible(B, Tq, Tk, len_q, len_k, causal, dev):
    """[B, 1, Tq, Tk]: which keys each query sees (queries of padding none)."""
    t, j = torch.arange(Tq, device=dev)[None, :, None], torch.arange(Tk, device=dev)[None, None]
    nq = torch.full((B,), Tq, device=dev) if len_q is None else len_q.long().clamp(0, Tq)
    nk = torch.full((B,), Tk, device=dev) if len_k is None else len_k.long().clamp(0, Tk)
    nq, nk = nq[:, None, None], nk[:, None, None]
    see = (t < nq) & (j < nk)
    if causal:
        see = see & (j <= t + nk - nq)
    return see[:, None]


def real(x, n):
    """x [B, H, T, D] in 64 bits with padding as 0."""
    x = x.double()
    if n is None:
        return x
    t = torch.arange(x.shape[2], device=x.device)
    return torch.where((t < n.long()[:, None])[:, None, :, None], x, 0.0)


def forward(q, k, v, gate=None, len_q=None, len_k=None, scale=None, causal=True):
    """o, lse and the bounds of their errors."""
    B, Hq, Tq, D = q.shape
    G, Tk = Hq // k.shape[1], k.shape[2]
    c = 1.0 / math.sqrt(D) if scale is None else scale
    q, k, v = real(q, len_q), heads(real(k, len_k), G), heads(real(v, len_k), G)
    see = visible(B, Tq, Tk, len_q, len_k, causal, q.device)
    s = torch.where(see, c * (q @ k.transpose(2, 3)), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(see, torch.exp(s - torch.where(lse > -math.inf, lse, 0.0)[..., None]), 0.0)
    sig = 1.0 if gate is None else torch.sigmoid(real(gate, len_q))
    es = torch.where(see, (D + 4) * 2.0 ** -23 * c * (q.abs() @ k.abs().transpose(2, 3)), 0.0)
    worst = es.amax(-1, keepdim=True) + 2.0 ** -22 * torch.where(lse > -math.inf, lse.abs(), 0.0)[..., None]
    o = (p @ v) * sig
    mag = p @ v.abs()
    bound = U * (mag * sig + o.abs()) + (2 * torch.expm1(2 * worst) + (Tk + 8) * 2.0 ** -23) * mag * sig + \
        Tk * 2.0 ** -24 * v.abs().amax((2, 3), keepdim=True) + 2.0 ** -25
    return o, lse, bound, worst[..., 0] + (Tk + 8) * 2.0 ** -23


def backward(do, q, k, v, o, lse, gate=None, len_q=None, len_k=None, scale=None, causal=True):
    """dq, dk, dv, dgate and the bounds of their errors, from the given o and lse."""
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    G = Hq // Hkv
    c = 1.0 / math.sqrt(D) if scale is None else scale
    q, do, o = real(q, len_q), real(do, len_q), real(o, len_q)
    k, v = heads(real(k, len_k), G), heads(real(v, len_k), G)
    see = visible(B, Tq, Tk, len_q, len_k, causal, q.device)
    lse = lse.double()
    finite = torch.where(see.any(-1), lse, 0.0)[..., None]
    p = torch.where(see, torch.exp(torch.where(see, c * (q @ k.transpose(2, 3)), 0.0) - finite), 0.0)
    sig = torch.ones_like(do) if gate is None else torch.sigmoid(real(gate, len_q))
    g, d = do * sig, (do * o).sum(-1, keepdim=True)
    dg, eg = do * o * (1 - sig), (U if gate is not None else 0.0) * g.abs() + (2.0 ** -25 if gate is not None else 0.0)
    dp = torch.where(see, g @ v.transpose(2, 3), 0.0)
    ds = torch.where(see, p * (dp - d), 0.0)
    group = lambda x: x.view(B, Hkv, G, *x.shape[2:]).sum(2)  # noqa: E731
    dv, dq, dk = group(p.transpose(2, 3) @ g), c * (ds @ k), c * group(ds.transpose(2, 3) @ q)
    # the errors of P and dS, element by element
    es = (D + 4) * 2.0 ** -23 * c * (q.abs() @ k.abs().transpose(2, 3)) + 2.0 ** -22 * finite.abs()
    rel = torch.expm1(2 * es)
    most = g.norm(dim=-1).amax() * v.norm(dim=-1).amax() + d.abs().amax()
    floor_p = max(2.0 ** -40, float(most) * 2.0 ** -38)
    ep = torch.where(see, p * (U + rel) + floor_p, 0.0)
    edp = (D + 4) * 2.0 ** -23 * (g.abs() @ v.abs().transpose(2, 3)) + eg @ v.abs().transpose(2, 3) + \
        (D + 4) * 2.0 ** -23 * (do * o).abs().sum(-1, keepdim=True)
    eds = torch.where(see, ds.abs() * (2 * U + rel) + ep * edp + p * edp + floor_p * (dp - d).abs() + float(most) * 2.0 ** -38, 0.0)
    n = (max(Tq * G, Tk) + 8) * 2.0 ** -23
    bv = group(ep.transpose(2, 3) @ g.abs() + (p + ep).transpose(2, 3) @ eg + n * (p.transpose(2, 3) @ g.abs()))
    bq = c * (eds @ k.abs() + n * (ds.abs() @ k.abs()))
    bk = c * group(eds.transpose(2, 3) @ q.abs() + n * (ds.abs().transpose(2, 3) @ q.abs()))
    out = lambda x, b: b * 1.01 + U * (x.abs() + b) + 2.0 ** -25  # noqa: E731
    return {"dq": dq, "dk": dk, "dv": dv, "dg": dg}, {"dq": out(dq, bq), "dk": out(dk, bk), "dv": out(dv, bv), "dg": out(dg, dg.abs() * 2.0 ** -20)}


def freqs(rot, base=10000.0, scaling=None, factor=1.0, orig_len=0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0):
    """Radians of one position for each pair, and amp."""
    out = []
    for i in range(rot // 2):
        b = base * factor ** (rot / (rot - 2)) if scaling == "ntk" else base
        f = b ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        if scaling == "yarn":
            lo = max(math.floor(rot * math.log(orig_len / (beta_fast * 2 * math.pi)) / (2 * math.log(base))), 0)
            hi = min(math.ceil(rot * math.log(orig_len / (beta_slow * 2 * math.pi)) / (2 * math.log(base))), rot - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f * (1 - r) + f / factor * r
        if scaling == "wavelength":
            keep = min(max((orig_len * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = f * keep + f / factor * (1 - keep)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64), 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


def rotate(x, pos, f, amp, interleaved, back=False):
    """x [B, H, T, D] at positions [B, T], in 64 bits."""
    R = 2 * f.numel()
    angle = pos.double()[:, None, :, None] * f.to(x.device)
    c, s = amp * torch.cos(angle), amp * torch.sin(angle) * (-1 if back else 1)
    y = x.double().clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def rotate_bound(x, y, pos, f, amp, interleaved):
    """Errors: the angle's (2^-65 turns a position, from the table, and this oracle's own 2^-52 of the
    angle), sine and cosine 2^-22 of 1, two products and a sum 2^-23 each, one rounding of the type."""
    R = 2 * f.numel()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    e = torch.zeros_like(y)
    angle = pos.double().abs()[:, None, :, None] * (f.to(x.device) * 2.0 ** -51 + 2 * math.pi * 2.0 ** -65)
    m = amp * (x[..., a].double().abs() + x[..., b].double().abs()) * (angle + 2.0 ** -22 + 2.0 ** -22)
    e[..., a], e[..., b] = m, m
    half = torch.finfo(x.dtype).eps / 2
    e[..., :R] += half * (y[..., :R].abs() + e[..., :R]) + (2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -149)
    return e
