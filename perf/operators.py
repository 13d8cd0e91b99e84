"""The 8-bit K/V cache and the attention that reads it, as a program that serves a model calls
them, beside their plain forms.

A case is a dict of plain values; `kind` names the operator:

  write    tsa.kv8_write of T new tokens per sequence, then tsa.kv8_read of the blocks they touch
  read     tsa.kv8_read of whole sequences
  attend   tsa.attn_kv8_fwd: T queries per sequence over its cache
  sparse   tsa.kv8_select, then tsa.attn_kv8_blocks_fwd over the selected blocks

The cache holds blocks of 64 tokens.  A full block's keys (and values) of one K/V head are 8-bit
codes with one scale: a = max|x|, code = round(127 x / a), value = code * a / 127.  The tokens
behind the last full block are fp16.  `len` counts each sequence's tokens, the new ones among
them; `ragged` sequences have lengths of their own.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 64


def listed():
    return [
        # one new token of one sequence, the gated grouped layer's K/V heads: latency counts
        {"name": "write_step_b1_d256", "kind": "write", "B": 1, "Hkv": 4, "D": 256, "T": 1, "len": 1000, "ragged": False},
        # one new token for each slot of a server, some of them filling a block
        {"name": "write_step_b48_d128", "kind": "write", "B": 48, "Hkv": 8, "D": 128, "T": 1, "len": 4111, "ragged": True},
        # two long prompts written at once: bandwidth
        {"name": "write_prompt_t8192_d256", "kind": "write", "B": 2, "Hkv": 4, "D": 256, "T": 8192, "len": 8192, "ragged": False},
        # short sequences of odd lengths handed to another consumer
        {"name": "read_b3_len2001_d64", "kind": "read", "B": 3, "Hkv": 2, "D": 64, "len": 2001, "ragged": True},
        # a long sequence read back whole
        {"name": "read_b1_len131072_d256", "kind": "read", "B": 1, "Hkv": 4, "D": 256, "len": 131072, "ragged": False},
        # one token of one chat over its history, the gated grouped layer: latency counts
        {"name": "decode_b1_len4097_d256", "kind": "attend", "B": 1, "Hq": 24, "Hkv": 4, "D": 256, "T": 1, "len": 4097, "ragged": False, "gate": True, "causal": True},
        # one token for each slot of a busy server with long contexts: bandwidth
        {"name": "decode_b32_len32768_d256", "kind": "attend", "B": 32, "Hq": 24, "Hkv": 4, "D": 256, "T": 1, "len": 32768, "ragged": True, "gate": True, "causal": True},
        # a few drafted tokens checked at once on a small model, odd lengths
        {"name": "verify_b8_t5_len2777_d64", "kind": "attend", "B": 8, "Hq": 16, "Hkv": 2, "D": 64, "T": 5, "len": 2777, "ragged": True, "gate": False, "causal": True},
        # a piece of a long prompt over what is cached of it
        {"name": "chunk_t512_len16384_d256", "kind": "attend", "B": 1, "Hq": 24, "Hkv": 4, "D": 256, "T": 512, "len": 16384, "ragged": False, "gate": True, "causal": True},
        # a whole prompt with equal query and K/V heads: the largest amount of arithmetic
        {"name": "prompt_t8192_h32_d128", "kind": "attend", "B": 1, "Hq": 32, "Hkv": 32, "D": 128, "T": 8192, "len": 8192, "ragged": False, "gate": False, "causal": True},
        # one token for each of 8 very long contexts, 32 of 2048 blocks each
        {"name": "sparse_step_b8_len131072_d256", "kind": "sparse", "B": 8, "Hq": 24, "Hkv": 4, "D": 256, "T": 1, "len": 131072, "ragged": True, "top": 32},
        # a piece of a long prompt, each query with blocks of its own
        {"name": "sparse_chunk_t700_len20001_d256", "kind": "sparse", "B": 1, "Hq": 24, "Hkv": 4, "D": 256, "T": 700, "len": 20001, "ragged": False, "top": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend", "sparse", "sparse"])
    D = rng.choice([64, 128, 256])
    ragged = rng.random() < 0.6
    if kind == "write":
        Hkv = rng.choice([1, 2, 4, 8, 32])
        if rng.random() < 0.5:  # a step: one token, or a few
            T, B = rng.choice([1, 1, 1, 2, 5, 17]), _log_int(rng, 1, 64)
            length = _log_int(rng, T + 1, 20000)
        else:  # a prompt, or a piece of one behind whole blocks
            T = _log_int(rng, 65, 8192)
            B = _log_int(rng, 1, max(1, 2 * 4 * 256 * 8192 // (Hkv * D * T)))
            length = T + BLOCK * rng.choice([0, 0, 1, 7])
        return {"kind": kind, "B": B, "Hkv": Hkv, "D": D, "T": T, "len": length, "ragged": ragged}
    if kind == "read":
        length, Hkv = _log_int(rng, 3, 131072), rng.choice([1, 2, 3, 4])
        B = _log_int(rng, 1, max(1, min(64, 4 * 256 * 131072 // (Hkv * D * length))))
        return {"kind": kind, "B": B, "Hkv": Hkv, "D": D, "len": length, "ragged": ragged}
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 3, 5, 6, 8, 12])
    if kind == "attend":
        if rng.random() < 0.5:  # single tokens, or a few
            T = rng.choice([1, 1, 1, 2, 4, 7])
            length = _log_int(rng, T, 65536)
            B = _log_int(rng, 1, max(1, min(64, 4 * 256 * 524288 // (Hkv * D * length))))
        else:
            T = _log_int(rng, 8, 4096)
            length = T + rng.choice([0, 0, 1, 64, 777, 4096])
            most = 32 * 8192 * 4096 * 128 // (D * Hkv * T * length)
            G = max(1, min(G, most))
            B = _log_int(rng, 1, max(1, min(8, most // G)))
        return {"kind": kind, "B": B, "Hq": Hkv * G, "Hkv": Hkv, "D": D, "T": T, "len": length, "ragged": ragged,
                "gate": rng.random() < 0.5, "causal": rng.random() < 0.8}
    top = rng.choice([4, 7, 16, 32, 64])
    if rng.random() < 0.6:
        T, B = rng.choice([1, 1, 2, 3]), _log_int(rng, 1, max(1, 32 // Hkv))
        length = _log_int(rng, 200, 131072 if B * Hkv <= 16 else 65536)
    else:
        T, B = _log_int(rng, 8, 700), 1
        top, Hkv = min(top, 16), min(Hkv, 4)
        length = T + _log_int(rng, 1, 20000)
    return {"kind": kind, "B": B, "Hq": Hkv * min(G, 8), "Hkv": Hkv, "D": D, "T": T, "len": length, "ragged": ragged, "top": top}


# Blocks that a sparse query keeps whatever they score: the first one, its own, and the two before it.
FIRST, RECENT = 1, 2


def _lens(case):
    """Each sequence's length and its number of new tokens (of T rows; behind them the rows are padding)."""
    B, L, T = case["B"], case["len"], case.get("T", 0)
    lens, new = [], []
    for b in range(B):
        n = T
        if case["ragged"] and b and T > 1:
            n = max(1, T - (b * 37) % T)
        cut = (b * 7919) % max(1, L // 2) if case["ragged"] else 0
        length = max(L - cut, n, 1)
        if case["kind"] == "write" and T > BLOCK:  # a prompt's piece starts behind whole blocks
            length = (L - T) + n
        lens.append(length)
        new.append(n)
    return lens, new


# ---------------------------------------------------------------------------------------
# the cache in its plain form: codes, scales and the open block's rows
# ---------------------------------------------------------------------------------------
def _quantise(x):
    """x [..., 64, D] fp16, whole blocks: codes int8 and the scale [...] of each block, in 32 bits."""
    x = x.float()
    a = x.abs().amax((-1, -2)).clamp_min(2.0 ** -24)
    return torch.round(127.0 * x / a[..., None, None]).to(torch.int8), a / torch.full_like(a, 127.0)


def _plain_cache(x, lens):
    """The cache of x [B, H, nb * 64, D] (rows behind a sequence's length are 0): codes [B, H, nb, 64, D],
    scales [B, H, nb], the open block's rows [B, H, 64, D]."""
    B, H, S, D = x.shape
    blocks = x.view(B, H, S // BLOCK, BLOCK, D)
    parts = [_quantise(blocks[:, h]) for h in range(H)]
    codes = torch.stack([p[0] for p in parts], 1)
    scale = torch.stack([p[1] for p in parts], 1)
    at = (lens.long() // BLOCK).clamp_max(S // BLOCK - 1)
    return codes, scale, blocks[torch.arange(B, device=x.device), :, at]


def _values(codes, scale, tail, lens):
    """The values [B, H, nb * 64, D] in 32 bits that a plain cache stands for."""
    B, H, nb, _, D = codes.shape
    x = codes.float() * scale[..., None, None]
    is_open = torch.arange(nb, device=codes.device) == (lens.long() // BLOCK)[:, None]
    x = torch.where(is_open[:, None, :, None, None], tail[:, :, None].float(), x)
    return x.view(B, H, nb * BLOCK, D)


def _summary(codes, scale):
    """A block's keys in one row: the sum of its codes, in 8 bits with a scale of its own."""
    c = codes.sum(-2, dtype=torch.int32).float()
    most = c.abs().amax(-1).clamp_min(1.0)
    return torch.round(127.0 * c / most[..., None]), (scale * most) * torch.full_like(most, 1.0 / (BLOCK * 127))


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _keys(case, S, gen, dev):
    """Keys and values [B, Hkv, S, D] fp16 as projections give them: channels of unequal size, and the
    keys of a block near each other."""
    B, H, D = case["B"], case["Hkv"], case["D"]
    rn = lambda *s: torch.randn(*s, generator=gen, device=dev, dtype=torch.float16)  # noqa: E731
    k = rn(B, H, S, D)
    k.view(B, H, S // BLOCK, BLOCK, D).add_(rn(B, H, S // BLOCK, 1, D))
    k.mul_(torch.exp(0.4 * rn(1, H, 1, D)))
    v = rn(B, H, S, D).mul_(torch.exp(0.3 * rn(1, H, 1, D)))
    return k, v


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    B, Hkv, D, T = case["B"], case["Hkv"], case["D"], case.get("T", 0)
    lens, new = _lens(case)
    S = -(-case["len"] // BLOCK) * BLOCK
    st = {"case": case, "max_len": case["len"]}
    st["len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["new"] = torch.tensor(new, dtype=torch.int32, device=dev) if T and min(new) < T else None
    k, v = _keys(case, S, gen, dev)
    rows = torch.arange(S, device=dev)
    behind = (rows >= st["len"][:, None])[:, None, :, None]
    k.masked_fill_(behind, 0)
    v.masked_fill_(behind, 0)
    held = st["len"]
    if case["kind"] == "write":  # the cache holds what came before the new tokens
        n_new = torch.tensor(new, dtype=torch.int32, device=dev)
        held = st["len"] - n_new
        t = torch.arange(T, device=dev)
        at = (held[:, None] + t).clamp_max(S - 1).long()[:, None, :, None].expand(B, Hkv, T, D)
        st["k"], st["v"] = k.gather(2, at), v.gather(2, at)
        st["start"] = held // BLOCK * BLOCK
        n = max(-(-ln // BLOCK) * BLOCK - (ln - m) // BLOCK * BLOCK for ln, m in zip(lens, new))
        st["k_out"], st["v_out"] = (torch.zeros(B, Hkv, n, D, dtype=torch.float16, device=dev) for _ in range(2))
        st["n_new"] = n_new
    if case["kind"] == "read":
        st["k_out"], st["v_out"] = (torch.zeros(B, Hkv, case["len"], D, dtype=torch.float16, device=dev) for _ in range(2))
    if case["kind"] in ("attend", "sparse"):
        st["q"] = torch.randn(B, case["Hq"], T, D, generator=gen, device=dev, dtype=torch.float16)
        st["gate"] = None
        if case.get("gate"):
            st["gate"] = torch.randn(B, case["Hq"], T, D, generator=gen, device=dev, dtype=torch.float16)
        st["out"] = torch.zeros_like(st["q"])
    if own:
        import_tsa()
        cache = st["cache"] = tsa.Kv8Cache(B, Hkv, D, max_len=S, device=dev)
        if int(held.max()) > 0:
            tsa.kv8_write(cache, k, v, held, held)
        if case["kind"] in ("attend", "sparse"):
            n = tsa.kv8_workspace_bytes(cache, T, case["Hq"], case["len"], case.get("top", 0))
            st["ws"] = torch.empty(n, dtype=torch.uint8, device=dev)
        if case["kind"] == "sparse":
            st["blocks"] = torch.full((B, Hkv, T, case["top"]), -1, dtype=torch.int32, device=dev)
    elif case["kind"] == "write":  # the open block's rows alone: full blocks are not read again
        st["cache"] = _plain_cache(k, held)[2], _plain_cache(v, held)[2]
    else:
        st["cache"] = _plain_cache(k, held), _plain_cache(v, held)
        if case["kind"] == "sparse":
            st["summary"] = _summary(*st["cache"][0][:2])
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
    if own:
        cache = st["cache"]
        if kind == "write":
            tsa.kv8_write(cache, st["k"], st["v"], st["len"], st["new"])
            tsa.kv8_read(cache, st["len"], start=st["start"], k_out=st["k_out"], v_out=st["v_out"])
            return {"k": st["k_out"], "v": st["v_out"]}
        if kind == "read":
            tsa.kv8_read(cache, st["len"], k_out=st["k_out"], v_out=st["v_out"])
            return {"k": st["k_out"], "v": st["v_out"]}
        if kind == "attend":
            tsa.attn_kv8_fwd(st["q"], cache, st["len"], st["new"], gate=st["gate"], out=st["out"], causal=case["causal"],
                             max_len=st["max_len"], ws=st["ws"])
            return {"o": st["out"]}
        tsa.kv8_select(st["q"], cache, st["len"], case["top"], st["new"], first=FIRST, recent=RECENT, out=st["blocks"],
                       max_len=st["max_len"], ws=st["ws"])
        tsa.attn_kv8_blocks_fwd(st["q"], cache, st["len"], st["blocks"], st["new"], out=st["out"], ws=st["ws"])
        return {"o": st["out"], "blocks": st["blocks"]}
    if kind == "write":
        return {"k": _plain_write(st, st["k"], st["cache"][0], st["k_out"]), "v": _plain_write(st, st["v"], st["cache"][1], st["v_out"])}
    if kind == "read":
        S = case["len"]
        inside = (torch.arange(S, device=st["len"].device) < st["len"][:, None])[:, None, :, None]
        k, v = (torch.where(inside, _values(*c, st["len"])[:, :, :S], 0.0).half() for c in st["cache"])
        return {"k": k, "v": v}
    return _plain_attend(st, case) if kind == "attend" else _plain_sparse(st, case)


def _plain_write(st, new, tail, like):
    """The touched blocks' values after the write: the open block's rows, the new ones behind them, and
    what became a full block through its codes."""
    B, H, n, D = like.shape
    T = new.shape[2]
    pos = st["start"][:, None] + torch.arange(n, device=new.device)
    old = (st["len"] - st["n_new"])[:, None]
    from_new = (pos - old).clamp(0, T - 1).long()[:, None, :, None].expand(B, H, n, D)
    from_tail = (pos % BLOCK).long()[:, None, :, None].expand(B, H, n, D)
    x = torch.where((pos < old)[:, None, :, None], tail.gather(2, from_tail), new.gather(2, from_new))
    inside = (pos < st["len"][:, None])[:, None, :, None]
    x = torch.where(inside, x.float(), 0.0)
    codes, scale = _quantise(x.view(B, H, n // BLOCK, BLOCK, D))
    full = ((pos // BLOCK + 1) * BLOCK <= st["len"][:, None])[:, None, :, None]
    return torch.where(full, (codes.float() * scale[..., None, None]).view(B, H, n, D), x).half()


def _places(st, T):
    """Each query's position [B, T], and whether its row is one (behind n_new they are padding)."""
    t = torch.arange(T, device=st["len"].device)
    new = st["new"] if st["new"] is not None else torch.full_like(st["len"], T)
    return (st["len"] - new)[:, None] + t, t < new[:, None]


def _plain_attend(st, case):
    q, Hkv = st["q"], case["Hkv"]
    B, Hq, T, D = q.shape
    k, v = (_values(*c, st["len"]) for c in st["cache"])
    S = k.shape[2]
    p, is_row = _places(st, T)
    s = torch.matmul(q.float().view(B, Hkv, -1, D), k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(B, Hkv, Hq // Hkv, T, S)
    j = torch.arange(S, device=q.device)
    hidden = j >= st["len"][:, None, None]
    if case["causal"]:
        hidden = hidden | (j > p[..., None])
    s.masked_fill_(hidden[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s.view(B, Hkv, -1, S), v).view(B, Hkv, Hq // Hkv, T, D) / s.sum(-1, keepdim=True)
    o = o.view(B, Hq, T, D)
    if st["gate"] is not None:
        o = o / (1.0 + torch.exp(-st["gate"].float()))
    return {"o": torch.where(is_row[:, None, :, None], o, 0.0).half()}


def _plain_sparse(st, case):
    q, Hkv, top = st["q"], case["Hkv"], case["top"]
    B, Hq, T, D = q.shape
    G = Hq // Hkv
    p, is_row = _places(st, T)
    qs = q.float().view(B, Hkv, G, T, D)
    # the cheap score: 8-bit queries of a group against 8-bit block summaries
    a = qs.abs().amax((2, 4), keepdim=True).clamp_min(2.0 ** -24)
    qc = torch.round(127.0 * qs / a)
    m, m_scale = st["summary"]
    nb = m.shape[2]
    score = torch.matmul(qc.view(B, Hkv, -1, D), m.transpose(2, 3)).view(B, Hkv, G, T, nb).amax(2) * m_scale[:, :, None]
    mine = (p // BLOCK)[:, None, :, None]
    i = torch.arange(nb, device=q.device)
    score = torch.where((i < FIRST) | (i >= mine - RECENT), math.inf, score)
    score = torch.where(i > mine, -math.inf, score)
    if nb < top:
        score = torch.cat([score, score.new_full((B, Hkv, T, top - nb), -math.inf)], -1)
    picked = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    picked = torch.where(picked > mine, 1 << 30, picked).sort(-1).values
    held = (picked < (1 << 30)) & is_row[:, None, :, None]
    at = torch.where(held, picked, 0)
    # attention of each query over its blocks
    bi, hi = torch.arange(B, device=q.device)[:, None, None, None], torch.arange(Hkv, device=q.device)[:, None, None]

    def gather(c):
        codes, scale, tail = c
        x = codes[bi, hi, at].float() * scale[bi, hi, at][..., None, None]
        is_open = at == (st["len"].long() // BLOCK)[:, None, None, None]
        return torch.where(is_open[..., None, None], tail[:, :, None, None].float(), x).view(B, Hkv, T, top * BLOCK, D)

    j = (at[..., None] * BLOCK + torch.arange(BLOCK, device=q.device)).view(B, Hkv, T, 1, top * BLOCK)
    hidden = (j > p[:, None, :, None, None]) | ~held[..., None].expand(B, Hkv, T, top, BLOCK).reshape(j.shape)
    qt = qs.transpose(2, 3)
    s = torch.matmul(qt, gather(st["cache"][0]).transpose(3, 4)).mul_(1.0 / math.sqrt(D))
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s, gather(st["cache"][1])) / s.sum(-1, keepdim=True)
    o = torch.where(is_row[:, None, :, None, None], o, 0.0).transpose(2, 3).reshape(B, Hq, T, D).half()
    return {"o": o, "blocks": torch.where(held, picked, -1).int()}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    B, Hkv, D, T = case["B"], case["Hkv"], case["D"], case.get("T", 0)
    lens, new = _lens(case)
    head = 2 * Hkv * D  # elements of one token's keys and values
    if case["kind"] == "write":
        # new rows in, full blocks' codes or the open rows out, and the touched blocks' values read back
        touched = sum(n + (ln - n) % BLOCK for ln, n in zip(lens, new))
        closed = sum(max(0, ln // BLOCK - (ln - n) // BLOCK) * BLOCK for ln, n in zip(lens, new))
        kept = sum(min(n, ln % BLOCK) for ln, n in zip(lens, new))
        return {"bytes": head * (2 * sum(new) + closed + 2 * kept + 2 * touched), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": head * sum(3 * (ln // BLOCK * BLOCK) + 4 * (ln % BLOCK) for ln in lens), "flops": 0}
    Hq = case["Hq"]
    io = sum(new) * Hq * D * 2 * (3 if case.get("gate") else 2)
    if case["kind"] == "attend":
        seen = lambda ln, n: n * ln - (n * (n - 1) // 2 if case["causal"] else 0)  # noqa: E731
        return {"bytes": io + head * sum(lens), "flops": 4 * Hq * D * sum(seen(ln, n) for ln, n in zip(lens, new))}
    blocks = [-(-ln // BLOCK) for ln in lens]
    listed_keys = [min(nb, case["top"]) * BLOCK for nb in blocks]
    summaries = Hkv * D * sum(blocks)
    read = head * sum(min(ln, n * keys) for ln, n, keys in zip(lens, new, listed_keys))
    flops = sum(n * Hq * D * (2 * nb + 4 * keys) for n, nb, keys in zip(new, blocks, listed_keys))
    return {"bytes": io + summaries + read, "flops": flops}


# ---------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------
def _exact_block_values(x, n_full):
    """x [n, D] float64 of one head: the values that the cache holds, full blocks through their codes.
    Also the codes and steps of the full blocks."""
    full = x[: n_full * BLOCK].reshape(n_full, BLOCK * x.shape[1])
    a = full.abs().max(1, keepdim=True).values if n_full else full.sum(1, keepdim=True)
    codes = torch.where(a > 0, torch.round(full * 127 / torch.where(a > 0, a, 1.0)), 0.0)
    values = (codes * (a / 127)).reshape(n_full * BLOCK, x.shape[1])
    return torch.cat([values, x[n_full * BLOCK:]]), codes.reshape(n_full, BLOCK, x.shape[1]), a[:, 0]


def exact(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    B, Hkv, D, T = case["B"], case["Hkv"], case["D"], case.get("T", 0)
    lens, new = _lens(case)
    k, v = _keys(case, -(-case["len"] // BLOCK) * BLOCK, gen, dev)
    f64 = {"dtype": torch.float64, "device": dev}
    if case["kind"] in ("write", "read"):
        starts = [(ln - n) // BLOCK * BLOCK if T else 0 for ln, n in zip(lens, new)]
        rows = max(-(-ln // BLOCK) * BLOCK - s for ln, s in zip(lens, starts)) if T else case["len"]
        found = {}
        for name, x in (("k", k), ("v", v)):
            out = found[name] = torch.zeros(B, Hkv, rows, D, **f64)
            for b in range(B):
                for h in range(Hkv):
                    got = _exact_block_values(x[b, h, starts[b]:lens[b]].double(), (lens[b] - starts[b]) // BLOCK)[0]
                    out[b, h, : len(got)] = got
        return found
    Hq = case["Hq"]
    G = Hq // Hkv
    q = torch.randn(B, Hq, T, D, generator=gen, device=dev, dtype=torch.float16)
    gate = torch.randn(B, Hq, T, D, generator=gen, device=dev, dtype=torch.float16) if case.get("gate") else None
    o = torch.zeros(B, Hq, T, D, **f64)
    for b in range(B):
        n, length = new[b], lens[b]
        pos = torch.arange(length - n, length, device=dev)
        for h in range(Hkv):
            kk, codes, a = _exact_block_values(k[b, h, :length].double(), length // BLOCK)
            vv = _exact_block_values(v[b, h, :length].double(), length // BLOCK)[0]
            group = q[b, h * G:(h + 1) * G, :n].double()
            may = torch.ones(n, length, dtype=torch.bool, device=dev)
            if case.get("causal", True):
                may = torch.arange(length, device=dev) <= pos[:, None]
            if case["kind"] == "sparse":
                chosen = _exact_choice(group, codes, a, pos, -(-length // BLOCK), case["top"])
                may = may & chosen.repeat_interleave(BLOCK, 1)[:, :length]
            for g in range(G):
                x = group[g] @ kk.T / math.sqrt(D)
                x = torch.where(may, x, -math.inf)
                w = torch.exp(x - x.max(1, keepdim=True).values)
                y = (w @ vv) / w.sum(1, keepdim=True)
                if gate is not None:
                    y = y * torch.sigmoid(gate[b, h * G + g, :n].double())
                o[b, h * G + g, :n] = y
    return {"o": o, "blocks": None} if case["kind"] == "sparse" else {"o": o}


def _exact_choice(group, codes, a, pos, nb, top):
    """The blocks [n, nb] that each query of a group keeps.  The score is a 32-bit number by definition:
    whole numbers, then one product with the block's 32-bit step."""
    n_full = codes.shape[0]
    big = group.abs().amax((0, 2), keepdim=True)
    qc = torch.round(group * 127 / torch.where(big > 0, big, 1.0))
    c = codes.sum(1)
    most = c.abs().max(1).values.clamp_min(1.0) if n_full else a
    m = torch.round(c * 127 / most[:, None])
    a = a.float().clamp_min(2.0 ** -24)
    step = a / torch.full_like(a, 127.0) * most.float() * torch.full_like(a, 1.0 / (BLOCK * 127))
    score = torch.full((len(pos), nb), -math.inf, dtype=torch.float32, device=codes.device)
    score[:, :n_full] = torch.stack([x @ m.T for x in qc]).max(0).values.float() * step
    mine, i = pos[:, None] // BLOCK, torch.arange(nb, device=codes.device)
    score[((i < FIRST) | (i >= mine - RECENT)).expand_as(score)] = math.inf
    score[(i > mine).expand_as(score)] = -math.inf
    order = torch.argsort(score, dim=1, descending=True, stable=True)[:, :top]
    chosen = torch.zeros(len(pos), nb, dtype=torch.bool, device=codes.device)
    chosen.scatter_(1, order, True)
    return chosen & (i <= mine)
