"""Rotary positions, attention's forward pass that keeps its row statistics and the backward pass that
reads them, as a program that serves or trains a model calls them, beside their plain forms.

A case is a dict of plain values; `kind` names the operator:

  rope   tsa.rope_fwd of a step's or a prompt's queries and keys, or tsa.rope_bwd of their gradients
  fwd    tsa.attn_train_fwd: gated grouped attention, and the logarithm of each row's softmax sum
  bwd    tsa.attn_bwd: the gradients of queries, keys, values and gate from what the forward left
  layer  one training step of an attention layer: the four calls in turn

Sequences of a padded batch (`ragged`) have lengths of their own; rows behind them hold numbers that no
result may depend on, and outputs there stay as they were (0 here).  Where a case has more keys than
queries (S > T), the queries are the last tokens.  `layout` is "bhsd" (a head's rows together) or
"bshd" (a token's heads together, as a projection leaves them).
"""
import math
import os
import sys

import torch

own = False


def listed():
    return [
        # one new token of one chat, the gated grouped layer's heads, a quarter of each rotated: latency counts
        {"name": "rope_step_b1_d256", "kind": "rope", "B": 1, "T": 1, "Hq": 24, "Hk": 4, "D": 256, "rot": 64, "pairs": "half", "type": "f16",
         "scaling": "none", "base": 1e6, "len": 4097, "ragged": False, "packed": False, "grad": False, "layout": "bhsd"},
        # one new token for each slot of a server with contexts stretched to 131072
        {"name": "rope_step_b48_d128", "kind": "rope", "B": 48, "T": 1, "Hq": 32, "Hk": 8, "D": 128, "rot": 128, "pairs": "half", "type": "f16",
         "scaling": "yarn", "base": 1e4, "len": 131072, "ragged": True, "packed": False, "grad": False, "layout": "bshd"},
        # a long prompt with equal query and key heads: bandwidth
        {"name": "rope_prompt_t8192_d128", "kind": "rope", "B": 1, "T": 8192, "Hq": 32, "Hk": 32, "D": 128, "rot": 128, "pairs": "interleaved",
         "type": "f16", "scaling": "none", "base": 1e4, "len": 8192, "ragged": False, "packed": False, "grad": False, "layout": "bshd"},
        # gradients of short documents packed into rows of odd length, in 32 bits
        {"name": "rope_grad_b3_t2001_d64", "kind": "rope", "B": 3, "T": 2001, "Hq": 16, "Hk": 2, "D": 64, "rot": 32, "pairs": "half", "type": "f32",
         "scaling": "wavelength", "base": 5e5, "len": 2001, "ragged": False, "packed": True, "grad": True, "layout": "bhsd"},
        # a padded batch of a small model, odd lengths
        {"name": "fwd_b5_t777_d64", "kind": "fwd", "B": 5, "T": 777, "S": 777, "Hq": 12, "Hkv": 4, "D": 64, "ragged": True, "gate": False,
         "causal": True, "layout": "bshd"},
        # the gated grouped layer over a long sequence
        {"name": "fwd_t8192_d256", "kind": "fwd", "B": 1, "T": 8192, "S": 8192, "Hq": 24, "Hkv": 4, "D": 256, "ragged": False, "gate": True,
         "causal": True, "layout": "bhsd"},
        # the lab's small shape without a mask: latency counts
        {"name": "bwd_t256_h4_d128", "kind": "bwd", "B": 1, "T": 256, "S": 256, "Hq": 4, "Hkv": 4, "D": 128, "ragged": False, "gate": False,
         "causal": False, "layout": "bhsd"},
        # the end of each sequence trained over what is in front of it, a padded batch of odd lengths
        {"name": "bwd_b3_t701_s1999_d256", "kind": "bwd", "B": 3, "T": 701, "S": 1999, "Hq": 6, "Hkv": 2, "D": 256, "ragged": True, "gate": True,
         "causal": True, "layout": "bshd"},
        # the gated grouped layer: few key heads, each with the sums of six query heads
        {"name": "bwd_t4096_d256", "kind": "bwd", "B": 1, "T": 4096, "S": 4096, "Hq": 24, "Hkv": 4, "D": 256, "ragged": False, "gate": True,
         "causal": True, "layout": "bshd"},
        # the lab's long shape: the largest amount of arithmetic
        {"name": "bwd_t8192_h32_d128", "kind": "bwd", "B": 1, "T": 8192, "S": 8192, "Hq": 32, "Hkv": 32, "D": 128, "ragged": False, "gate": False,
         "causal": True, "layout": "bhsd"},
        # a step of a small model's layer
        {"name": "layer_b2_t512_d64", "kind": "layer", "B": 2, "T": 512, "S": 512, "Hq": 8, "Hkv": 8, "D": 64, "ragged": False, "gate": False,
         "causal": True, "layout": "bshd", "rot": 64, "pairs": "half", "scaling": "none", "base": 1e4},
        # a step of a grouped layer on a padded batch
        {"name": "layer_b4_t2048_d128", "kind": "layer", "B": 4, "T": 2048, "S": 2048, "Hq": 32, "Hkv": 8, "D": 128, "ragged": True, "gate": True,
         "causal": True, "layout": "bshd", "rot": 64, "pairs": "interleaved", "scaling": "linear", "base": 1e4},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rope(rng, D):
    rot = rng.choice([D, D, D // 2, D // 4, D // 8 * 3, 20 if D == 64 else 32])
    return {"rot": rot, "pairs": rng.choice(["half", "interleaved"]), "base": rng.choice([1e4, 5e5, 1e6]),
            "scaling": rng.choice(["none", "none", "linear", "ntk", "yarn", "wavelength"])}


def draw(rng):
    kind = rng.choice(["rope", "rope", "rope", "fwd", "fwd", "bwd", "bwd", "bwd", "bwd", "layer"])
    D = rng.choice([64, 128, 256])
    layout = rng.choice(["bhsd", "bshd"])
    Hkv, G = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 6, 8])
    if kind == "rope":
        kinds = rng.choice(["step", "prompt", "train"])
        most = 8192 * 64 * 128 // (Hkv * (G + 1) * D)  # tokens in all
        if kinds == "step":
            B, T = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 5])
        else:
            T = _log_int(rng, 3, min(most, 16384))
            B = _log_int(rng, 1, max(1, min(16, most // T)))
        return {"kind": kind, "B": B, "T": T, "Hq": Hkv * G, "Hk": Hkv, "D": D, **_draw_rope(rng, D), "type": rng.choice(["f16", "f16", "f32"]),
                "len": T + _log_int(rng, 1, 200000) if kinds == "step" else T, "ragged": B > 1 and rng.random() < 0.5,
                "packed": kinds == "train" and rng.random() < 0.7, "grad": kinds == "train", "layout": layout}
    # attention: the work of the largest listed case at most, 32 heads of 8192 x 8192 / 2 x 128
    causal = rng.random() < 0.75
    most = 32 * 8192 * 8192 * 128 // (2 if causal else 4)
    T = _log_int(rng, 1, 4096)
    S = T if kind == "layer" or rng.random() < 0.6 else T + _log_int(rng, 1, 4096)
    while T * S * D * Hkv * G > most:
        Hkv, G = max(1, Hkv // 2), max(1, G // 2)
        if Hkv * G == 1:
            break
    B = _log_int(rng, 1, max(1, min(16, most // (T * S * D * Hkv * G))))
    case = {"kind": kind, "B": B, "T": T, "S": S, "Hq": Hkv * G, "Hkv": Hkv, "D": D, "ragged": B > 1 and rng.random() < 0.6,
            "gate": rng.random() < 0.5, "causal": causal, "layout": layout}
    if kind == "layer":
        case.update(_draw_rope(rng, D))
    return case


# The parameters of the scaled frequencies, one set for each kind.
FACTOR, ORIG_LEN, BETA_FAST, BETA_SLOW, LOW, HIGH = 8.0, 16384, 32.0, 1.0, 1.0, 4.0


def _lens(case):
    """Queries and keys of each sequence."""
    B, T, S = case["B"], case["T"], case.get("S", case["T"])
    if not case["ragged"]:
        return [T] * B, [S] * B
    lq = [max(1, T - (b * 7919) % max(1, T)) for b in range(B)]
    lk = list(lq) if S == T else [max(n, S - (b * 4567) % S) for b, n in enumerate(lq)]
    return lq, lk


def _counts(case):
    """A step's tokens after the call, and its new tokens, of each sequence."""
    lq, _ = _lens(case)
    return [n + max(0, (case["len"] - case["T"]) - (b * 50021 if case["ragged"] else 0) % max(1, case["len"] - case["T"] + 1)) for b, n in enumerate(lq)], lq


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _normal(case, H, rows, gen, dtype=torch.float16):
    """[B, H, rows, D] in the case's layout."""
    shape = (case["B"], H, rows, case["D"]) if case["layout"] == "bhsd" else (case["B"], rows, H, case["D"])
    x = torch.randn(*shape, generator=gen, device=gen.device, dtype=dtype)
    return x if case["layout"] == "bhsd" else x.transpose(1, 2)


def _outliers(x, gen):
    """One element of a hundred eight times as large, as activations have them."""
    return x.mul_(torch.where(torch.rand(x.shape, generator=gen, device=x.device) < 0.01, 8.0, 1.0).to(x.dtype))


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    st = {"case": case}
    B, T = case["B"], case["T"]
    if case["kind"] == "rope":
        dtype = torch.float32 if case["type"] == "f32" else torch.float16
        st["q"], st["k"] = _normal(case, case["Hq"], T, gen, dtype), _normal(case, case["Hk"], T, gen, dtype)
        if case["packed"]:  # documents one behind the other: positions begin again
            starts = torch.rand(B, T, generator=gen, device=dev) < 0.004
            starts[:, 0] = True
            t = torch.arange(T, device=dev).expand(B, T)
            st["pos"] = (t - torch.where(starts, t, 0).cummax(1).values).int()
        return st, gen
    S, Hq, Hkv = case["S"], case["Hq"], case["Hkv"]
    st["q"] = _outliers(_normal(case, Hq, T, gen).mul_(0.7), gen)
    st["k"] = _outliers(_normal(case, Hkv, S, gen).mul_(0.7), gen)
    st["v"] = _normal(case, Hkv, S, gen)
    st["gate"] = _normal(case, Hq, T, gen) if case["gate"] else None
    if case["kind"] != "fwd":  # a token's gradient is larger or smaller as a whole
        st["do"] = _normal(case, Hq, T, gen).mul_(0.1 * torch.exp(torch.randn(B, 1, T, 1, generator=gen, device=dev))).half()
    return st, gen


def _like(x):
    return torch.zeros_like(x, memory_format=torch.preserve_format)


def _set_up(st):
    """Lengths and, for the backward pass, what the forward pass left."""
    case, dev = st["case"], st["q"].device
    lq, lk = _lens(case)
    if case["kind"] == "rope":
        if not case["packed"]:
            counts, new = _counts(case)
            st["len"] = torch.tensor(counts, dtype=torch.int32, device=dev)
        st["new"] = torch.tensor(lq, dtype=torch.int32, device=dev) if case["ragged"] else None
        return
    st["lq"], st["lk"] = (torch.tensor(x, dtype=torch.int32, device=dev) if case["ragged"] else None for x in (lq, lk))
    if case["kind"] == "bwd":
        st["o"], st["lse"] = _plain_fwd(st["q"], st["k"], st["v"], st["gate"], st["lq"], st["lk"], case["causal"])


def prepare(case, seed):
    st, _ = _inputs(case, seed)
    _set_up(st)
    kind = case["kind"]
    q, k = st["q"], st["k"]
    if kind == "rope":
        st["q_out"], st["k_out"] = _like(q), _like(k)
    else:
        v = st["v"]
        if kind != "bwd":
            st["o_out"] = _like(q)
            st["lse_out"] = torch.zeros(q.shape[:3], dtype=torch.float32, device=q.device)
        if kind != "fwd":
            st["dq"], st["dk"], st["dv"] = _like(q), _like(k), _like(v)
            st["dg"] = _like(q) if case["gate"] else None
        if kind == "layer":
            st["q_rot"], st["k_rot"], st["dq_rot"], st["dk_rot"] = _like(q), _like(k), _like(q), _like(k)
    if own:
        import_tsa()
        if kind in ("rope", "layer"):
            scaling = {} if case["scaling"] == "none" else {"scaling": case["scaling"], "factor": FACTOR, "orig_len": ORIG_LEN,
                                                            "beta_fast": BETA_FAST, "beta_slow": BETA_SLOW, "low": LOW, "high": HIGH}
            st["rope"] = tsa.Rope(case["D"], rot=case["rot"], base=case["base"], interleaved=case["pairs"] == "interleaved", **scaling)
        if kind in ("bwd", "layer"):
            n = tsa.attn_bwd_workspace_bytes(case["B"], case["Hq"], case["Hkv"], case["T"], case["S"], case["D"], gated=case["gate"],
                                             causal=case["causal"])
            st["ws"] = torch.empty(n, dtype=torch.uint8, device=q.device)
    elif kind in ("rope", "layer"):
        st["freq"], st["amp"] = _plain_freq(case, q.device)
    return st


def import_tsa():
    global tsa
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "turing-sm75_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tsa as module
    tsa = module


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    kind = case["kind"]
    q, k = st["q"], st["k"]
    if kind == "rope":
        if own:
            fn = tsa.rope_bwd if case["grad"] else tsa.rope_fwd
            fn(st["rope"], q, k, pos=st.get("pos"), len=st.get("len"), n_new=st["new"], q_out=st["q_out"], k_out=st["k_out"])
            return {"q": st["q_out"], "k": st["k_out"]}
        pos = st["pos"] if case["packed"] else _positions(st, q.shape[2])
        rows = st["new"]
        return {"q": _plain_rope(q, pos, st, case["grad"], rows), "k": _plain_rope(k, pos, st, case["grad"], rows)}
    v, gate, lq, lk, causal = st["v"], st["gate"], st["lq"], st["lk"], case["causal"]
    if own:
        if kind == "layer":
            tsa.rope_fwd(st["rope"], q, k, n_new=lq, q_out=st["q_rot"], k_out=st["k_rot"])
            q, k = st["q_rot"], st["k_rot"]
        if kind != "bwd":
            o, lse = tsa.attn_train_fwd(q, k, v, gate, len_q=lq, len_k=lk, out=st["o_out"], lse=st["lse_out"], causal=causal)
        if kind == "fwd":
            return {"o": o, "lse": lse}
        if kind == "bwd":
            o, lse = st["o"], st["lse"]
        dq, dk = (st["dq_rot"], st["dk_rot"]) if kind == "layer" else (st["dq"], st["dk"])
        tsa.attn_bwd(st["do"], q, k, v, o, lse, gate, len_q=lq, len_k=lk, dq=dq, dk=dk, dv=st["dv"], dgate=st["dg"], causal=causal, ws=st["ws"])
        if kind == "layer":
            tsa.rope_bwd(st["rope"], dq, dk, n_new=lq, q_out=st["dq"], k_out=st["dk"])
        found = {"dq": st["dq"], "dk": st["dk"], "dv": st["dv"]}
        if gate is not None:
            found["dg"] = st["dg"]
        return {**found, "o": o} if kind == "layer" else found
    if kind == "layer":
        pos = torch.arange(q.shape[2], device=q.device).expand(q.shape[0], -1)
        q, k = _plain_rope(q, pos, st, False, lq), _plain_rope(k, pos, st, False, lq)
    if kind != "bwd":
        o, lse = _plain_fwd(q, k, v, gate, lq, lk, causal)
    if kind == "fwd":
        return {"o": o, "lse": lse}
    if kind == "bwd":
        o, lse = st["o"], st["lse"]
    dq, dk, dv, dg = _plain_bwd(st["do"], q, k, v, o, lse, gate, lq, lk, causal)
    if kind == "layer":
        dq, dk = _plain_rope(dq, pos, st, True, lq), _plain_rope(dk, pos, st, True, lq)
    found = {"dq": dq, "dk": dk, "dv": dv}
    if gate is not None:
        found["dg"] = dg
    return {**found, "o": o} if kind == "layer" else found


# ---------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------
def _plain_freq(case, dev):
    """Angles of one position, in 64 bits, and the factor on the rotated elements."""
    R, base, kind = case["rot"], case["base"], case["scaling"]
    i = torch.arange(R // 2, device=dev, dtype=torch.float64)
    if kind == "ntk":
        base = base * FACTOR ** (R / (R - 2))
    f = base ** (-2.0 * i / R)
    if kind == "linear":
        return f / FACTOR, 1.0
    if kind == "yarn":  # pairs that turn often within the original length stay, slow ones are stretched
        turns_at = lambda n: R * math.log(ORIG_LEN / (n * 2.0 * math.pi)) / (2.0 * math.log(base))  # noqa: E731
        low, high = max(math.floor(turns_at(BETA_FAST)), 0), min(math.ceil(turns_at(BETA_SLOW)), R - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f * (1.0 - ramp) + f / FACTOR * ramp, 0.1 * math.log(FACTOR) + 1.0
    if kind == "wavelength":  # turns within the original length: many stay, few are stretched, linear between
        turns = ORIG_LEN * f / (2.0 * math.pi)
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0.0, 1.0)
        return f * keep + f / FACTOR * (1.0 - keep), 1.0
    return f, 1.0


def _positions(st, T):
    new = st["new"] if st["new"] is not None else torch.full_like(st["len"], T)
    return (st["len"] - new)[:, None] + torch.arange(T, device=new.device)


def _plain_rope(x, pos, st, grad, rows):
    R, amp = st["case"]["rot"], st["amp"]
    angle = pos.double()[:, None, :, None] * st["freq"]
    cos, sin = (torch.cos(angle) * amp).float(), (torch.sin(angle) * (-amp if grad else amp)).float()
    y = x.float().clone(memory_format=torch.preserve_format)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if st["case"]["pairs"] == "interleaved" else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = xa * cos - xb * sin
    y[..., b] = xb * cos + xa * sin
    if rows is not None:
        y = torch.where(torch.arange(x.shape[2], device=x.device)[None, None, :, None] < rows[:, None, None, None], y, 0.0)
    return y.to(x.dtype)


def _pieces(q, S):
    """Slices of (sequence, head) pairs whose scores take 1 GiB at most."""
    B, H, T, _ = q.shape
    n = max(1, (1 << 28) // (T * S))
    return [(i, min(B * H, i + n)) for i in range(0, B * H, n)]


def _hidden(q, S, lq, lk, causal, at):
    """[pairs, T, S]: keys that a query does not see (queries of padding see none)."""
    B, H, T, _ = q.shape
    dev = q.device
    b = torch.arange(*at, device=dev) // H
    t, j = torch.arange(T, device=dev)[None, :, None], torch.arange(S, device=dev)[None, None]
    nq = (lq[b] if lq is not None else torch.full_like(b, T))[:, None, None]
    nk = (lk[b] if lk is not None else torch.full_like(b, S))[:, None, None]
    return (j >= nk) | (t >= nq) | (j > t + nk - nq if causal else j < 0)


def _rows(x, at, group):
    """Rows [pairs, ., D] in 32 bits of the heads that these pairs of sequence and query head read."""
    B, H = x.shape[:2]
    i = torch.arange(*at, device=x.device) // group
    return x[i // H, i % H].float()


def _plain_fwd(q, k, v, gate, lq, lk, causal):
    B, H, T, D = q.shape
    S, G = k.shape[2], H // k.shape[1]
    o, lse = torch.zeros(B * H, T, D, device=q.device), torch.zeros(B * H, T, device=q.device)
    for at in _pieces(q, S):
        s = torch.matmul(_rows(q, at, 1), _rows(k, at, G).transpose(1, 2)).mul_(1.0 / math.sqrt(D))
        s.masked_fill_(_hidden(q, S, lq, lk, causal, at), -math.inf)
        m = s.amax(-1, keepdim=True).clamp_min(-3e38)
        p = s.sub_(m).exp_()
        total = p.sum(-1, keepdim=True)
        o[at[0]:at[1]] = torch.matmul(p, _rows(v, at, G)) / total.clamp_min(1e-30)
        lse[at[0]:at[1]] = torch.where(total > 0, torch.log(total) + m, -math.inf)[..., 0]
    o, lse = o.view(B, H, T, D), lse.view(B, H, T)
    if gate is not None:
        o = o / (1.0 + torch.exp(-gate.float()))
    if lq is not None:
        lse = torch.where(torch.arange(T, device=q.device) < lq[:, None, None], lse, 0.0)
    return o.half(), lse


def _plain_bwd(do, q, k, v, o, lse, gate, lq, lk, causal):
    B, H, T, D = q.shape
    Hkv, S = k.shape[1:3]
    G = H // Hkv
    scale = 1.0 / math.sqrt(D)
    g, dg = do.float(), None
    is_row = None if lq is None else torch.arange(T, device=q.device)[None, None, :, None] < lq[:, None, None, None]
    delta = (g * o.float()).sum(-1)
    if gate is not None:
        sig = 1.0 / (1.0 + torch.exp(-gate.float()))
        dg = g * o.float() * (1.0 - sig)
        dg = (dg if is_row is None else torch.where(is_row, dg, 0.0)).half()
        g = g * sig
    delta, lse = delta.reshape(B * H, T, 1), lse.reshape(B * H, T, 1)
    dq = torch.zeros(B * H, T, D, device=q.device)
    dk, dv = torch.zeros(B * Hkv, S, D, device=q.device), torch.zeros(B * Hkv, S, D, device=q.device)
    for at in _pieces(q, S):
        rows = slice(*at)
        qq, kk, vv, gg = _rows(q, at, 1), _rows(k, at, G), _rows(v, at, G), _rows(g, at, 1)
        p = torch.matmul(qq, kk.transpose(1, 2)).mul_(scale).sub_(lse[rows]).exp_()
        hidden = _hidden(q, S, lq, lk, causal, at)
        p.masked_fill_(hidden, 0.0)
        if is_row is not None:
            gg.masked_fill_(~is_row[torch.arange(*at, device=q.device) // H, 0], 0.0)
        heads = torch.arange(*at, device=q.device) // G
        dv.index_add_(0, heads, torch.matmul(p.transpose(1, 2), gg))
        ds = torch.matmul(gg, vv.transpose(1, 2)).sub_(delta[rows]).mul_(p).masked_fill_(hidden, 0.0)
        dq[rows] = torch.matmul(ds, kk).mul_(scale)
        dk.index_add_(0, heads, torch.matmul(ds.transpose(1, 2), qq).mul_(scale))
    return dq.view(B, H, T, D).half(), dk.view(B, Hkv, S, D).half(), dv.view(B, Hkv, S, D).half(), dg


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    B, T, D = case["B"], case["T"], case["D"]
    lq, lk = _lens(case)
    n = sum(lq)
    if case["kind"] == "rope":
        return {"bytes": 2 * n * (case["Hq"] + case["Hk"]) * D * (4 if case["type"] == "f32" else 2) + (4 * n if case["packed"] else 0), "flops": 0}
    Hq, Hkv, gate = case["Hq"], case["Hkv"], int(case["gate"])
    pairs = Hq * sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(lq, lk))
    row, keys = 2 * D * Hq * n, 2 * D * Hkv * sum(lk)
    stat = 4 * Hq * n
    fwd = {"bytes": row * (2 + gate) + 2 * keys + stat, "flops": 4 * D * pairs}
    bwd = {"bytes": row * (4 + 2 * gate) + 4 * keys + stat, "flops": 10 * D * pairs}
    if case["kind"] == "fwd":
        return fwd
    if case["kind"] == "bwd":
        return bwd
    # the layer: every input once (q, k, v, gate, dO), every output once (o, dq, dk, dv, dg)
    return {"bytes": row * (4 + 2 * gate) + 4 * keys, "flops": 14 * D * pairs}


# ---------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------
def _exact_angles(case, pos):
    """[n, R / 2] angles of positions, and the factor on what is rotated."""
    R, s = case["rot"], FACTOR
    out, amp = [], 1.0
    for i in range(R // 2):
        f = math.exp(-2.0 * i / R * math.log(case["base"]))
        if case["scaling"] == "linear":
            f /= s
        elif case["scaling"] == "ntk":
            f = math.exp(-2.0 * i / R * (math.log(case["base"]) + R / (R - 2) * math.log(s)))
        elif case["scaling"] == "yarn":
            bound = [R * math.log(ORIG_LEN / (2 * math.pi * beta)) / (2 * math.log(case["base"])) for beta in (BETA_FAST, BETA_SLOW)]
            lo, hi = max(math.floor(bound[0]), 0), min(math.ceil(bound[1]), R - 1)
            part = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f, amp = f * (part / s + 1 - part), 1 + 0.1 * math.log(s)
        elif case["scaling"] == "wavelength":
            part = min(max((ORIG_LEN / (2 * math.pi / f) - LOW) / (HIGH - LOW), 0.0), 1.0)
            f = part * f + (1 - part) * f / s
        out.append(f)
    return pos[:, None] * torch.tensor(out, dtype=torch.float64, device=pos.device), amp


def _exact_rope(x, case, pos, sign):
    """x [H, n, D] float64 at positions [n] (float64)."""
    R = case["rot"]
    angle, amp = _exact_angles(case, pos)
    z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) if case["pairs"] == "interleaved" else torch.complex(x[..., : R // 2], x[..., R // 2:R])
    z = z * torch.polar(torch.full_like(angle, amp), sign * angle)
    y = x.clone()
    if case["pairs"] == "interleaved":
        y[..., :R] = torch.stack([z.real, z.imag], -1).flatten(-2)
    else:
        y[..., :R] = torch.cat([z.real, z.imag], -1)
    return y


def _stored(x):
    """What one call of a layer's step leaves for the next is held in 16 bits."""
    return x.half().double()


def exact(case, seed):
    st, _ = _inputs(case, seed)
    dev = st["q"].device
    B, T, D = case["B"], case["T"], case["D"]
    f64 = {"dtype": torch.float64, "device": dev}
    lq, lk = _lens(case)
    if case["kind"] == "rope":
        found = {name: torch.zeros(st[name].shape, **f64) for name in ("q", "k")}
        counts = None if case["packed"] else _counts(case)[0]
        for b in range(B):
            n = lq[b]
            pos = st["pos"][b, :n].double() if case["packed"] else torch.arange(counts[b] - n, counts[b], **f64)
            for name in found:
                found[name][b, :, :n] = _exact_rope(st[name][b, :, :n].double(), case, pos, -1.0 if case["grad"] else 1.0)
        return found
    _set_up(st)
    Hq, Hkv, S = case["Hq"], case["Hkv"], case["S"]
    G, scale = Hq // Hkv, 1.0 / math.sqrt(D)
    whole = {name: torch.zeros(B, Hq, T, D, **f64) for name in ("o", "dq", "dg")}
    whole.update({name: torch.zeros(B, Hkv, S, D, **f64) for name in ("dk", "dv")})
    whole["lse"] = torch.zeros(B, Hq, T, **f64)
    for b in range(B):
        n, m = lq[b], lk[b]
        see = None
        if case["causal"]:
            see = torch.arange(m, device=dev)[None] <= (torch.arange(n, device=dev) + (m - n))[:, None]
        pos = torch.arange(n, **f64)
        for h in range(Hq):
            q, k, v = st["q"][b, h, :n].double(), st["k"][b, h // G, :m].double(), st["v"][b, h // G, :m].double()
            if case["kind"] == "layer":
                q, k = (_stored(_exact_rope(x[None], case, pos, 1.0)[0]) for x in (q, k))
            s = (q @ k.T) * scale
            if see is not None:
                s = torch.where(see, s, -math.inf)
            sig = torch.sigmoid(st["gate"][b, h, :n].double()) if case["gate"] else torch.ones(n, D, **f64)
            if case["kind"] == "bwd":  # the statistics and the output are inputs
                lse, o = st["lse"][b, h, :n].double(), st["o"][b, h, :n].double()
                p = torch.exp(s - lse[:, None])
            else:
                lse = torch.logsumexp(s, 1)
                p = torch.exp(s - lse[:, None])
                o = (p @ v) * sig
                whole["o"][b, h, :n], whole["lse"][b, h, :n] = o, lse
                o = _stored(o)
            if case["kind"] == "fwd":
                continue
            do = st["do"][b, h, :n].double()
            whole["dg"][b, h, :n] = do * o * (1.0 - sig)
            z = do * sig
            whole["dv"][b, h // G, :m] += p.T @ z
            p *= (z @ v.T) - (do * o).sum(1, keepdim=True)
            whole["dq"][b, h, :n], dk = (p @ k) * scale, (p.T @ q) * scale
            whole["dk"][b, h // G, :m] += dk
        if case["kind"] == "layer":
            for name in ("dq", "dk"):
                whole[name][b, :, :n] = _exact_rope(_stored(whole[name][b, :, :n]), case, pos, -1.0)
    names = {"fwd": ["o", "lse"], "bwd": ["dq", "dk", "dv"], "layer": ["dq", "dk", "dv", "o"]}[case["kind"]]
    return {name: whole[name] for name in names + (["dg"] if case["gate"] and case["kind"] != "fwd" else [])}
