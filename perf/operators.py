"""Speculative decoding over a long or quantised KV cache, as timed cases.

A step of it rotates the drafted tokens' queries and keys at their positions
("rope"), writes keys and values into a cache of 8-bit codes ("append"), reads
such a cache back where a prompt attends to it ("read"), attends with a tree of
drafted tokens, or one token, over the cache ("attn") and verifies the drafted
tokens against the target's probabilities ("verify").

`run` computes each in plain torch, or, with `own` set, through this
repository's entry points. Formulas:

rope    out = x turned, pair by pair, by the angle position * inv_freq[j] over
        the first `rotary` elements of a head, cos and sin times `factor`; the
        rest of a head, and tokens at negative positions, are copied
append  a cache row (one head of one token) is codes c and one exponent byte e,
        x ~ c * 2^(e - 127): the least power of two with max|x| <= M * 2^(e -
        127), M = 448 (e4m3) or 127 (int8), e in 1 .. 254; c = x / 2^(e - 127)
        rounded half to even
read    c * 2^(e - 127) in the model's type
attn    softmax(scale q k^T) v over the context's keys and, of the drafted
        tokens' keys that follow them in the cache, a token's ancestors and
        itself
verify  a chain with the draft's probabilities q: token i stays while u_i q_i <
        p_i, then one is drawn from max(p - q, 0), or from p behind the last; a
        tree: at each node one of its children, by inverse CDF over them, or
        none, then one drawn from p without the children
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
CODE_MAX = {"e4m3": 448.0, "int8": 127.0}
VOCAB, THETA = 151936, 1e6
# drawn cases stay at or below the largest listed case of their operator
MAX_ROPE = 4 * 4096 * 24 * 128         # elements turned
MAX_ROWS = 8 * 8 * 2304 * 128          # cache elements read or written, of K
MAX_KEYS = 32 * 8 * 2048 * 128         # cache elements attended to, of K
MAX_SCORES = 2 * 32 * 33 * 32768       # scores of one call
MAX_PROBS = 16 * 32 * 151936           # target probabilities


def listed():
    return [
        # the drafted tokens of eight sequences, at the depths of their trees
        {"name": "rope-draft-8x16", "op": "rope", "batch": 8, "seq": 16, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "rotary": 128, "interleaved": False, "scaling": 1.0, "far": 2048,
         "dtype": "bf16"},
        # a long prompt, half of each head rotated in interleaved pairs, the
        # positions scaled for a context four times the trained one
        {"name": "rope-prompt-4x4096", "op": "rope", "batch": 4, "seq": 4096, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "rotary": 64, "interleaved": True, "scaling": 4.0,
         "far": 120000, "dtype": "fp16"},
        # the drafted tokens' keys and values into the cache
        {"name": "append-draft-8x16", "op": "append", "codes": "int8", "batch": 8, "seq": 16,
         "kv_heads": 8, "head_dim": 128, "min_len": 900, "max_len": 2200, "capacity": 2304,
         "dtype": "bf16"},
        # a batch of prompts into the cache
        {"name": "append-prompt-8x2048", "op": "append", "codes": "e4m3", "batch": 8, "seq": 2048,
         "kv_heads": 8, "head_dim": 128, "min_len": 0, "max_len": 0, "capacity": 2304,
         "dtype": "bf16"},
        # the cached prefix of eight sequences, for the attention of a next prompt
        {"name": "read-8x2304", "op": "read", "codes": "e4m3", "batch": 8, "len": 2304,
         "kv_heads": 8, "head_dim": 128, "capacity": 2304, "dtype": "bf16"},
        # one conversation of odd length
        {"name": "read-1x777", "op": "read", "codes": "int8", "batch": 1, "len": 777,
         "kv_heads": 8, "head_dim": 64, "capacity": 1024, "dtype": "fp16"},
        # one token of one sequence, where latency counts
        {"name": "attn-token-1x700", "op": "attn", "codes": "int8", "batch": 1, "tokens": 1,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "min_len": 700, "max_len": 700,
         "capacity": 2304, "dtype": "bf16"},
        # one token each of a serving batch of mixed lengths
        {"name": "attn-token-32", "op": "attn", "codes": "e4m3", "batch": 32, "tokens": 1,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "min_len": 100, "max_len": 4096,
         "capacity": 8192, "dtype": "bf16"},
        # trees of sixteen drafted tokens over a 16-bit cache
        {"name": "attn-tree-8x16", "op": "attn", "codes": "none", "batch": 8, "tokens": 16,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "min_len": 1500, "max_len": 2288,
         "capacity": 2304, "dtype": "bf16"},
        # wide groups and trees over a long cache
        {"name": "attn-tree-2x33-long", "op": "attn", "codes": "e4m3", "batch": 2, "tokens": 33,
         "heads": 32, "kv_heads": 4, "head_dim": 128, "min_len": 20000, "max_len": 32700,
         "capacity": 32768, "dtype": "fp16"},
        # chains of five drafted tokens with the draft model's probabilities
        {"name": "verify-chain-8x5", "op": "verify", "kind": "chain", "batch": 8, "tokens": 5,
         "vocab": VOCAB, "filtered": False},
        # trees of the draft's best tokens, the target's rows cut to their nucleus
        {"name": "verify-tree-16x31", "op": "verify", "kind": "tree", "batch": 16, "tokens": 31,
         "vocab": VOCAB, "filtered": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attn", "attn", "attn", "verify", "verify"])
    case = {"op": op}
    if op != "verify":
        case["dtype"] = rng.choice(["fp16", "bf16"])
    if op == "rope":
        heads, head_dim = rng.choice([8, 12, 16, 32]), rng.choice([64, 80, 128, 256])
        batch = rng.choice([1, 2, 3, 4, 8])
        kv_heads = heads // rng.choice([1, 2, 4])
        case.update(batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    seq=max(1, min(_log(rng, 1, 8192), MAX_ROPE // (batch * (heads + kv_heads) * head_dim))),
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2, 32, 20]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice([1.0, 1.0, 4.0, 8.0]),
                    far=_log(rng, 16, 1000000))
    elif op in ("append", "read"):
        kv_heads, head_dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128])
        batch = _log(rng, 1, 32)
        room = MAX_ROWS // (batch * kv_heads * head_dim)
        capacity = min(rng.choice([256, 1024, 2304, 8192, 32768]), room // 16 * 16)
        seq = max(1, min(_log(rng, 1, capacity), capacity))
        case.update(codes=rng.choice(["e4m3", "int8"]), batch=batch, kv_heads=kv_heads,
                    head_dim=head_dim, capacity=capacity)
        if op == "read":
            case["len"] = seq
        else:
            far = rng.randint(0, capacity - seq)
            case.update(seq=seq, min_len=rng.randint(0, far), max_len=far)
    elif op == "attn":
        tokens = rng.choice([1, 1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
        heads, group = rng.choice([8, 16, 32]), rng.choice([1, 2, 4, 8])
        head_dim, kv_heads = rng.choice([64, 128]), heads // group
        batch = _log(rng, 1, 48)
        capacity = rng.choice([c for c in (512, 2304, 4096, 8192, 16384, 32768)
                               if kv_heads * c * head_dim <= MAX_KEYS])
        batch = max(1, min(batch, MAX_KEYS // (kv_heads * capacity * head_dim),
                           MAX_SCORES // (heads * tokens * capacity)))
        max_len = _log(rng, 16, capacity - tokens)
        case.update(codes=rng.choice(["none", "e4m3", "int8"]), batch=batch, tokens=tokens,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    min_len=rng.choice([max_len, _log(rng, 1, max_len)]), max_len=max_len,
                    capacity=capacity)
    else:
        vocab = rng.choice([VOCAB, VOCAB, 32000, 50257, 131072])
        tokens = _log(rng, 1, 48)
        case.update(kind=rng.choice(["chain", "chain", "tree"]), tokens=tokens, vocab=vocab,
                    batch=max(1, min(_log(rng, 1, 32), MAX_PROBS // ((tokens + 1) * vocab))),
                    filtered=rng.random() < 0.5)
    return case


# ---- what a program holds before the call ------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _tree(tokens, rs):
    """Parents (-1: the context) of a random tree in topological order, and
    its ancestor-or-self matrix."""
    parents = np.array([int(rs.randint(max(-1, t - 8), t)) for t in range(tokens)], dtype=np.int32)
    see = np.zeros((tokens, tokens), dtype=bool)
    for t in range(tokens):
        if parents[t] >= 0:
            see[t] = see[parents[t]]
        see[t, t] = True
    return parents, see


def _trees(batch, tokens, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    both = [_tree(tokens, rs) for _ in range(batch)]
    return (torch.from_numpy(np.stack([b[0] for b in both])).to(DEV),
            torch.from_numpy(np.stack([b[1] for b in both])).to(DEV))


def _lengths(case, gen):
    return torch.randint(case["min_len"], case["max_len"] + 1, (case["batch"],), generator=gen,
                         device=DEV, dtype=torch.int32)


def _codes(case, gen):
    """Codes and exponent bytes of keys (or values) of about unit size."""
    shape = (case["batch"], case["kv_heads"], case["capacity"], case["head_dim"])
    if case["codes"] == "e4m3":
        codes = (_randn(shape, gen) * 130).clamp(-448, 448).to(torch.float8_e4m3fn)
        e = torch.randint(118, 122, shape[:3], generator=gen, device=DEV, dtype=torch.uint8)
    else:
        codes = (_randn(shape, gen) * 40).clamp(-127, 127).round().to(torch.int8)
        e = torch.randint(120, 124, shape[:3], generator=gen, device=DEV, dtype=torch.uint8)
    return codes, e


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    st = {"case": dict(case)}
    if op == "rope":
        dt, b, s, d = TYPES[case["dtype"]], case["batch"], case["seq"], case["head_dim"]
        hq, hk = case["heads"], case["kv_heads"]
        qkv = _randn((b, s, (hq + 2 * hk) * d), gen, dt)  # a fused projection's output
        st["q"] = qkv[..., : hq * d].view(b, s, hq, d)
        st["k"] = qkv[..., hq * d : (hq + hk) * d].view(b, s, hk, d)
        start = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device=DEV)
        st["positions"] = (start + torch.arange(s, device=DEV)).int()
        j = torch.arange(0, case["rotary"], 2, device=DEV, dtype=torch.float64)
        st["inv_freq"] = THETA ** (-j / case["rotary"]) / case["scaling"]
        st["factor"] = 1.0 if case["scaling"] == 1.0 else 0.1 * math.log(case["scaling"]) + 1.0
    elif op == "append":
        dt = TYPES[case["dtype"]]
        b, s, h, d = case["batch"], case["seq"], case["kv_heads"], case["head_dim"]
        kv = _randn((b, s, 2 * h * d), gen)
        kv = (kv * torch.exp(_randn((b, s, 1), gen))).to(dt)  # rows of different sizes
        st["k"], st["v"] = (kv[..., i * h * d : (i + 1) * h * d].view(b, s, h, d) for i in (0, 1))
        st["positions"] = _lengths(case, gen)
        shape = (b, h, case["capacity"], d)
        for n in ("k", "v"):
            st[n + "_codes"] = torch.zeros(shape, device=DEV, dtype=CODES[case["codes"]])
            st[n + "_exps"] = torch.full(shape[:3], 127, device=DEV, dtype=torch.uint8)
    elif op == "read":
        for n in ("k", "v"):
            st[n + "_codes"], st[n + "_exps"] = _codes(case, gen)
    elif op == "attn":
        dt, b, t, d = TYPES[case["dtype"]], case["batch"], case["tokens"], case["head_dim"]
        st["q"] = _randn((b, t, case["heads"], d), gen, dt)
        st["lens"] = _lengths(case, gen)
        st["parents"], st["see"] = _trees(b, t, seed)
        if case["codes"] == "none":
            shape = (b, case["kv_heads"], case["capacity"], d)
            st["k"], st["v"] = _randn(shape, gen, dt), _randn(shape, gen, dt)
        else:
            for n in ("k", "v"):
                st[n + "_codes"], st[n + "_exps"] = _codes(case, gen)
    else:
        b, t, v = case["batch"], case["tokens"], case["vocab"]
        p = _randn((b, t + 1, v), gen).mul_(2.5)
        if case["kind"] == "chain":
            q = p[:, :t] + _randn((b, t, v), gen)  # the draft is near the target
            st["draft_probs"] = torch.softmax(q, -1)
            del q
        p = torch.softmax(p, -1)
        if case["filtered"]:
            p *= p >= p.amax(-1, keepdim=True) * 0.02
            p /= p.sum(-1, keepdim=True)
        st["target_probs"] = p
        st["uniforms"] = torch.rand((b, t + 1), generator=gen, device=DEV)
        if case["kind"] == "chain":
            rows = st["draft_probs"].view(b * t, v)
            st["tokens"] = torch.multinomial(rows, 1, generator=gen).view(b, t)
        else:
            st["parents"], st["see"] = _trees(b, t, seed)
            same = st["parents"].unsqueeze(2) == st["parents"].unsqueeze(1)  # [B, T, T]
            rank = (same & torch.ones_like(same).tril(-1)).sum(2)            # earlier siblings
            best = p.topk(int(rank.max()) + 1, -1).indices                   # [B, T + 1, .]
            row = (st["parents"].long() + 1).unsqueeze(2).expand(-1, -1, best.shape[2])
            st["tokens"] = best.gather(1, row).gather(2, rank.unsqueeze(2)).squeeze(2)
    return st


# ---- the plain forms ---------------------------------------------------------------


def _turn(x, cos, sin, rotary, interleaved):
    y = x.float()
    if interleaved:
        a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., : rotary // 2], y[..., rotary // 2 : rotary]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., rotary:]], -1).to(x.dtype)


def _rope(st):
    case = st["case"]
    ang = st["positions"].double().unsqueeze(-1) * st["inv_freq"]
    cos, sin = ((f(ang) * st["factor"]).float().unsqueeze(2) for f in (torch.cos, torch.sin))
    return {n: _turn(st[n], cos, sin, case["rotary"], case["interleaved"]) for n in ("q", "k")}


def _append(st):
    case = st["case"]
    most = CODE_MAX[case["codes"]]
    b, s = case["batch"], case["seq"]
    at = st["positions"].long().unsqueeze(1) + torch.arange(s, device=DEV)       # [B, S]
    seq = torch.arange(b, device=DEV).unsqueeze(1).expand(b, s)
    out = {}
    for n in ("k", "v"):
        x = st[n].float()
        frac, exp = torch.frexp(x.abs().amax(-1) / most)  # amax / M = frac 2^exp, frac in [1/2, 1)
        e = (exp - (frac == 0.5).int()).clamp(-126, 127)  # the least with amax <= M 2^e
        c = torch.ldexp(x, -e.unsqueeze(-1))
        c = c.round() if case["codes"] == "int8" else c
        codes = st[n + "_codes"]
        codes.view(torch.uint8)[seq, :, at] = c.to(codes.dtype).view(torch.uint8)
        st[n + "_exps"][seq, :, at] = (e + 127).to(torch.uint8)
        out[n + "_codes"], out[n + "_exps"] = st[n + "_codes"], st[n + "_exps"]
    return out


def _values(codes, exps):
    return torch.ldexp(codes.float(), exps.int().unsqueeze(-1) - 127)


def _read(st):
    n, dt = st["case"]["len"], TYPES[st["case"]["dtype"]]
    return {x: _values(st[x + "_codes"][:, :, :n], st[x + "_exps"][:, :, :n]).to(dt) for x in ("k", "v")}


def _attn(st):
    case, q = st["case"], st["q"]
    b, t, hq, d = q.shape
    hk, n = case["kv_heads"], case["max_len"] + t
    if case["codes"] == "none":
        k, v = st["k"][:, :, :n].float(), st["v"][:, :, :n].float()
    else:
        k, v = (_values(st[x + "_codes"][:, :, :n], st[x + "_exps"][:, :, :n]) for x in ("k", "v"))
    rows = q.float().view(b, t, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    s = torch.matmul(rows, k.transpose(2, 3)).mul_(d ** -0.5).view(b, hk, hq // hk, t, n)
    rel = torch.arange(n, device=DEV) - st["lens"].long().unsqueeze(1)           # [B, N]
    drafted = st["see"].gather(2, rel.clamp(0, t - 1).unsqueeze(1).expand(b, t, n))
    seen = (rel < 0).unsqueeze(1) | (drafted & (rel < t).unsqueeze(1))           # [B, T, N]
    s.masked_fill_(~seen.unsqueeze(1).unsqueeze(1), -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(e.view(b, hk, -1, n), v) / e.sum(-1).view(b, hk, -1, 1)
    return {"o": o.view(b, hk, hq // hk, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d).to(q.dtype)}


def _drawn(w, u):
    """First index at which the running sum of a row of weights passes u times
    the row's sum."""
    cum = w.cumsum(-1)
    return (cum > u.double().unsqueeze(-1) * cum[:, -1:]).int().argmax(-1)


def _verify(st):
    case, p, u, tok = st["case"], st["target_probs"], st["uniforms"], st["tokens"]
    b, t = tok.shape
    seq, nodes = torch.arange(b, device=DEV), torch.arange(t, device=DEV)
    if case["kind"] == "chain":
        q = st["draft_probs"]
        pt = p[:, :t].gather(2, tok.unsqueeze(2)).squeeze(2).double()
        qt = q.gather(2, tok.unsqueeze(2)).squeeze(2).double()
        stays = (u[:, :t].double() * qt < pt).int().cumprod(1)
        n = stays.sum(1)
        path = torch.where(stays.bool(), nodes, -1)
        row = p[seq, n].double()
        rest = (row - q[seq, n.clamp(max=t - 1)].double()).clamp(min=0)
        rest = torch.where((n < t).unsqueeze(1), rest, row)
    else:
        par = st["parents"].long()
        mass = p[seq.unsqueeze(1), par + 1, tok].double()  # of each node, in its parent's row
        earlier = (par.unsqueeze(2) == par.unsqueeze(1)) & (nodes.unsqueeze(1) > nodes)
        below = (earlier * mass.unsqueeze(1)).sum(2)
        depth = st["see"].sum(2) - 1
        ud = u.gather(1, depth).double()
        taken = (below <= ud) & (ud < below + mass)
        kept = taken & ~(st["see"] & ~taken.unsqueeze(1)).any(2)
        n = kept.sum(1)
        path = torch.where(kept, nodes, t).sort(1).values
        path = torch.where(path < t, path, -1)
        last = torch.where(kept, nodes, -1).amax(1)
        child = (par == last.unsqueeze(1)).int()
        out = torch.zeros(b, p.shape[2], device=DEV, dtype=torch.int32).scatter_add_(1, tok, child)
        row = p[seq, last + 1].double()
        rest = row * (out == 0)
    rest = torch.where((rest.sum(1) > 0).unsqueeze(1), rest, row)
    return {"accepted": n.int(), "path": path.int(), "next_token": _drawn(rest, u[:, t])}


# ---- the calls a user makes --------------------------------------------------------


def _own(st):
    case, op = st["case"], st["case"]["op"]
    if op == "rope":
        from torchplusplus_amd.dlops.rope import rope_apply_at
        q, k = rope_apply_at(st["q"], st["k"], st["positions"], st["inv_freq"],
                             interleaved=case["interleaved"], attention_factor=st["factor"])
        return {"q": q, "k": k}
    if op == "append":
        from torchplusplus_amd.llmops.kvcache import kv_quant_append
        kv_quant_append(st["k"], st["v"], st["k_codes"], st["v_codes"], st["k_exps"], st["v_exps"],
                        st["positions"])
        return {n: st[n] for n in ("k_codes", "k_exps", "v_codes", "v_exps")}
    if op == "read":
        from torchplusplus_amd.llmops.kvcache import kv_quant_read
        k, v = kv_quant_read(st["k_codes"], st["v_codes"], st["k_exps"], st["v_exps"], case["len"],
                             TYPES[case["dtype"]])
        return {"k": k, "v": v}
    if op == "attn":
        from torchplusplus_amd.attention import tree_attention
        if case["codes"] == "none":
            return {"o": tree_attention(st["q"], st["k"], st["v"], st["lens"], st["parents"])}
        return {"o": tree_attention(st["q"], st["k_codes"], st["v_codes"], st["lens"], st["parents"],
                                    k_exps=st["k_exps"], v_exps=st["v_exps"])}
    from torchplusplus_amd.llmops.speculative import verify_draft
    n, path, nxt = verify_draft(st["tokens"], st["target_probs"], st["uniforms"],
                                draft_probs=st.get("draft_probs"), parents=st.get("parents"))
    return {"accepted": n, "path": path, "next_token": nxt}


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope, "append": _append, "read": _read, "attn": _attn,
            "verify": _verify}[state["case"]["op"]](state)


# ---- what a pass cannot do without, and its result in 64 bits -------------------------


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 4 * n + 4 * case["batch"] * case["seq"], "flops": 3 * n}
    if op in ("append", "read"):
        rows = case["batch"] * case["kv_heads"] * case["seq" if op == "append" else "len"]
        return {"bytes": 2 * rows * (3 * case["head_dim"] + 1), "flops": 2 * rows * case["head_dim"]}
    if op == "attn":
        keys = case["batch"] * ((case["min_len"] + case["max_len"]) / 2 + case["tokens"])
        d, rows = case["head_dim"], case["tokens"] * case["heads"]
        row = 2 * d if case["codes"] == "none" else d + 1
        return {"bytes": 2 * keys * case["kv_heads"] * row + 4 * case["batch"] * rows * d,
                "flops": 4 * keys * rows * d}
    rows = case["batch"] * case["vocab"]
    return {"bytes": 4 * rows * (2 if case["kind"] == "chain" else 1), "flops": 2 * rows}


def exact(case, seed):
    op = case["op"]
    if op == "verify" or (op == "append" and case["codes"] == "int8"):
        return None  # whole numbers only
    st = prepare(case, seed)
    if op == "rope":
        out = {}
        half = case["rotary"] // 2
        for n in ("q", "k"):
            x = st[n].double()
            z = x.clone()
            for j in range(half):
                a = st["positions"].double() * st["inv_freq"][j]
                c, s = torch.cos(a).unsqueeze(2) * st["factor"], torch.sin(a).unsqueeze(2) * st["factor"]
                lo, hi = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
                z[..., lo] = x[..., lo] * c - x[..., hi] * s
                z[..., hi] = x[..., lo] * s + x[..., hi] * c
            out[n] = z
        return out
    if op == "append":
        out, most = {}, CODE_MAX[case["codes"]]
        for n in ("k", "v"):
            x = st[n].double()
            codes = torch.zeros(st[n + "_codes"].shape, dtype=torch.float64, device=DEV)
            e = torch.full(x.shape[:3], -126.0, dtype=torch.float64, device=DEV)
            amax = x.abs().amax(-1)
            for p in range(-126, 127):  # the least power that holds the row
                e[amax > most * 2.0 ** p] = p + 1
            y = x * torch.exp2(-e).unsqueeze(-1)
            step = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)
            y = (y / step).round() * step
            for i, at in enumerate(st["positions"].tolist()):
                codes[i, :, at : at + case["seq"]] = y[i].transpose(0, 1)
            out[n + "_codes"], out[n + "_exps"] = codes, None  # the exponents are whole numbers
        return out
    if op == "read":
        n = case["len"]
        return {x: st[x + "_codes"][:, :, :n].double()
                * torch.exp2(st[x + "_exps"][:, :, :n].double() - 127).unsqueeze(-1) for x in ("k", "v")}
    q, t = st["q"].double(), case["tokens"]
    o = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for i, n in enumerate(st["lens"].tolist()):
        see = torch.cat([torch.ones(t, n, dtype=torch.bool, device=DEV), st["see"][i]], 1)
        for h in range(case["kv_heads"]):
            if case["codes"] == "none":
                k, v = (st[x][i, h, : n + t].double() for x in ("k", "v"))
            else:
                k, v = (st[x + "_codes"][i, h, : n + t].double()
                        * torch.exp2(st[x + "_exps"][i, h, : n + t].double() - 127).unsqueeze(1)
                        for x in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                s = (q[i, :, g] @ k.T) / math.sqrt(case["head_dim"])
                s[~see] = -math.inf
                o[i, :, g] = torch.softmax(s, -1) @ v
    return {"o": o}
