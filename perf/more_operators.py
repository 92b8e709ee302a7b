"""Serving a mixed batch over a paged cache, as timed cases.

Prompts and turns of different lengths are packed one behind the other, each
attending to its own ("packed"); a step's projections are normed, rotated at
their tokens' positions and written into the pages of a cache ("write"); one new
token of every sequence attends to its pages ("paged"); and rows of logits give
the log probabilities of chosen tokens, the entropy and the best alternatives
("logprobs").

`run` computes each in plain torch, or, with `own` set, through this
repository's entry points. Formulas:

packed    o_i = softmax_j(q_i k_j / sqrt(D)) v_j over the keys j of i's own
          sequence with j <= i + Lk - Lq (and, in a window, j >= i + Lk - Lq - w)
write     head rows x of q and k: y = x / sqrt(mean(x^2) + eps) * w, then turned,
          y' = y cos(p) + rotate_half(y) sin(p); k's rows, and v's as they are, go
          to row slot % page_size of page slot / page_size
paged     o = softmax_j(q k_j / sqrt(D)) v_j over the first len keys, key j in row
          j % page_size of page table[j / page_size]
logprobs  x_t - log sum_j e^x_j of a token t, - sum_j p_j log p_j, and the same for
          the `top` largest logits, the lowest index first among equal ones
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB, THETA, EPS = 151936, 1e6, 1e-6
CONTEXT = 32768  # rows of the rotation's tables
# drawn cases stay at or below the largest listed case of their operator
MAX_PAIRS = 16 * 3.6e7                 # heads x visible (query, key) pairs
MAX_SCORES = 8 * 16 * 4096 * 4096      # scores of the plain form, every sequence as long as the longest
MAX_KEYS = 2 * 100000 * 4 * 128        # cache elements attended to, of K
MAX_PADDED = 32 * 4096 * 8 * 128       # the same with every sequence as long as the longest
MAX_ROWS = 16000 * 32 * 128            # elements of a projection
MAX_LOGITS = 1024 * 151936


def listed():
    return [
        # a serving batch of eight prompts, the shape of a prefill of this decoder
        {"name": "packed-prompts-8", "op": "packed", "batch": 8, "min_len": 501, "max_len": 4001,
         "prefix": 0, "window": -1, "heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # one short prompt, where latency counts
        {"name": "packed-one-230", "op": "packed", "batch": 1, "min_len": 230, "max_len": 230,
         "prefix": 0, "window": -1, "heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # sixty-four short requests of 3 to 200 tokens
        {"name": "packed-short-64", "op": "packed", "batch": 64, "min_len": 3, "max_len": 200,
         "prefix": 0, "window": -1, "heads": 16, "kv_heads": 16, "head_dim": 64, "dtype": "fp16"},
        # follow-up turns behind 2500 tokens each, in a sliding window
        {"name": "packed-turns-6", "op": "packed", "batch": 6, "min_len": 40, "max_len": 700,
         "prefix": 2500, "window": 1023, "heads": 32, "kv_heads": 4, "head_dim": 128, "dtype": "bf16"},
        # one token of one sequence
        {"name": "paged-1x700", "op": "paged", "batch": 1, "min_len": 700, "max_len": 700, "page": 16,
         "window": -1, "heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # one token each of a serving batch of mixed lengths
        {"name": "paged-32", "op": "paged", "batch": 32, "min_len": 100, "max_len": 4096, "page": 64,
         "window": -1, "heads": 16, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # two long documents, wide groups
        {"name": "paged-2-long", "op": "paged", "batch": 2, "min_len": 60000, "max_len": 100000, "page": 256,
         "window": -1, "heads": 32, "kv_heads": 4, "head_dim": 128, "dtype": "fp16"},
        # a decode step of 32 sequences
        {"name": "write-32", "op": "write", "tokens": 32, "page": 64, "norm": True, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # a packed batch of prompts
        {"name": "write-16000", "op": "write", "tokens": 16000, "page": 64, "norm": True, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # the tokens of one decode step, with the alternatives that an answer lists
        {"name": "logprobs-8", "op": "logprobs", "rows": 8, "vocab": VOCAB, "top": 5, "dtype": "bf16"},
        # a prompt of a thousand tokens scored
        {"name": "logprobs-1024", "op": "logprobs", "rows": 1024, "vocab": VOCAB, "top": 5, "dtype": "bf16"},
        # logits in fp32 over an odd vocabulary, many alternatives
        {"name": "logprobs-77-fp32", "op": "logprobs", "rows": 77, "vocab": 50257, "top": 20, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _pairs(case):
    """Visible (query, key) pairs of every sequence, of one head."""
    n = 0
    for length in _lengths(case):
        first = case["prefix"] + 1  # keys that the first query sees, without a window
        if case["window"] < 0:
            n += length * first + length * (length - 1) // 2
        else:
            most = case["window"] + 1
            short = min(length, max(0, most - first + 1))  # queries that see all keys up to their own
            n += short * first + short * (short - 1) // 2 + (length - short) * most
    return n


def draw(rng):
    while True:
        op = rng.choice(["packed", "packed", "packed", "paged", "paged", "paged", "write", "logprobs", "logprobs"])
        case = {"op": op, "dtype": rng.choice(["fp16", "bf16"])}
        if op in ("packed", "paged"):
            heads = rng.choice([8, 16, 32])
            max_len = _log(rng, 1, 6000 if op == "packed" else 60000)
            case.update(heads=heads, kv_heads=heads // rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128, 128]),
                        batch=_log(rng, 1, 64), min_len=rng.choice([max_len, _log(rng, 1, max_len)]),
                        max_len=max_len, window=rng.choice([-1, -1, -1, _log(rng, 16, 4096)]))
        if op == "packed":
            case["prefix"] = rng.choice([0, 0, 0, _log(rng, 1, 4000)])
            most = case["batch"] * case["max_len"] * (case["prefix"] + case["max_len"]) * case["heads"]
            if most > MAX_SCORES or _pairs(case) * case["heads"] * case["head_dim"] > MAX_PAIRS * 128:
                continue
        elif op == "paged":
            case["page"] = rng.choice([16, 32, 64, 128, 256])
            each = case["kv_heads"] * case["head_dim"]
            if sum(_lengths(case)) * each > MAX_KEYS or case["batch"] * max_len * each > MAX_PADDED:
                continue
        elif op == "write":
            heads = rng.choice([8, 12, 16, 32])
            case.update(heads=heads, kv_heads=heads // rng.choice([1, 2, 4]), head_dim=rng.choice([64, 128, 256]),
                        tokens=_log(rng, 1, 16000), page=rng.choice([16, 32, 64, 128, 256]), norm=rng.random() < 0.7)
            if case["tokens"] * (heads + 2 * case["kv_heads"]) * case["head_dim"] > MAX_ROWS:
                continue
        else:
            vocab = rng.choice([VOCAB, VOCAB, 32000, 50257, 131072, _log(rng, 100, 200000)])
            case.update(rows=_log(rng, 1, 4096), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]),
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            if case["rows"] * vocab * (2 if case["dtype"] == "fp32" else 1) > MAX_LOGITS:
                continue
        return case


# ---- what a program holds before the call ------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _lengths(case):
    """The sequences' lengths, evenly from the least to the most on a log scale."""
    n, lo, hi = case["batch"], case["min_len"], case["max_len"]
    return [round(lo * (hi / lo) ** (i / max(n - 1, 1))) for i in range(n)] if n > 1 else [hi]


def _shuffled(case, seed):
    x = _lengths(case)
    np.random.RandomState(seed % (1 << 31)).shuffle(x)
    return x


def _ends(lengths):
    return torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device=DEV)


def _tables(head_dim):
    """cos and sin of the rotation, [CONTEXT, D] fp16, as this repository's models keep them."""
    j = torch.arange(0, head_dim, 2, device=DEV, dtype=torch.float64)
    a = torch.arange(CONTEXT, device=DEV, dtype=torch.float64).unsqueeze(1) * THETA ** (-j / head_dim)
    a = torch.cat([a, a], 1)
    return torch.cos(a).half(), torch.sin(a).half()


def prepare(case, seed):
    gen, op, dt = _gen(seed), case["op"], TYPES[case["dtype"]]
    st = {"case": dict(case)}
    if op == "logprobs":
        st["logits"] = (_randn((case["rows"], case["vocab"]), gen) * 2.5).to(dt)
        st["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device=DEV)
        return st
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if op == "packed":
        st["lens"] = _shuffled(case, seed)
        n, nk = sum(st["lens"]), sum(st["lens"]) + case["prefix"] * case["batch"]
        st["q"] = _randn((n, hq, d), gen, dt)
        kv = _randn((nk, 2 * hk, d), gen, dt)
        st["k"], st["v"] = kv[:, :hk], kv[:, hk:]
        st["cu"], st["cu_k"] = _ends(st["lens"]), _ends([x + case["prefix"] for x in st["lens"]])
    elif op == "paged":
        st["lens"] = _shuffled(case, seed)
        st["seqlens"] = torch.tensor(st["lens"], dtype=torch.int32, device=DEV)
        each = [-(-x // case["page"]) for x in st["lens"]]
        total = sum(each)
        order = torch.randperm(total, generator=gen, device=DEV).int()
        table = torch.full((case["batch"], max(each)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, x in enumerate(each):
            table[i, :x] = order[at : at + x]
            at += x
        st["table"] = table
        st["q"] = _randn((case["batch"], hq, d), gen, dt)
        st["k_pages"] = _randn((total, hk, case["page"], d), gen, dt)
        st["v_pages"] = _randn((total, hk, case["page"], d), gen, dt)
    else:
        n, page = case["tokens"], case["page"]
        pages = -(-2 * n // page) + 1
        st["qkv"] = _randn((n, (hq + 2 * hk) * d), gen, dt)
        st["positions"] = torch.randint(0, CONTEXT, (n,), generator=gen, device=DEV, dtype=torch.int32)
        st["slots"] = torch.randperm(pages * page, generator=gen, device=DEV)[:n]
        for x in ("k_pages", "v_pages"):
            st[x] = torch.zeros((pages, hk, page, d), dtype=dt, device=DEV)
        for x in ("q_norm", "k_norm"):
            st[x] = (1 + 0.1 * _randn((d,), gen)).to(dt) if case["norm"] else None
        st["cos"], st["sin"] = _tables(d)
    return st


# ---- the plain forms ---------------------------------------------------------------


def _attend(q, k, v, seen):
    """q [B, Hk, G, Lq, D], k and v [B, Hk, Lk, D], seen [B, Lq, Lk]; 32 bits."""
    b, hk, g, n, d = q.shape
    s = torch.matmul(q.reshape(b, hk, g * n, d), k.transpose(2, 3)).mul_(d ** -0.5).view(b, hk, g, n, -1)
    s.masked_fill_(~seen.view(b, 1, 1, n, -1), -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    return (torch.matmul(s.view(b, hk, g * n, -1), v).view(b, hk, g, n, d) / total).nan_to_num_(0.0)


def _padded(x, ends, most):
    """Rows of [N, H, D] as [B, H, most, D], fp32; rows past a sequence's end are other sequences'."""
    at = (ends[:-1].long().unsqueeze(1) + torch.arange(most, device=DEV)).clamp_(max=x.shape[0] - 1)
    return x[at].float().transpose(1, 2).contiguous()


def _packed(st):
    case = st["case"]
    hk, n, nk = case["kv_heads"], case["max_len"], case["max_len"] + case["prefix"]
    q, k, v = _padded(st["q"], st["cu"], n), _padded(st["k"], st["cu_k"], nk), _padded(st["v"], st["cu_k"], nk)
    i = torch.arange(n, device=DEV).view(1, n, 1) + case["prefix"]
    j = torch.arange(nk, device=DEV).view(1, 1, nk)
    seen = j <= i
    if case["window"] >= 0:
        seen = seen & (j >= i - case["window"])
    o = _attend(q.view(len(st["lens"]), hk, -1, n, q.shape[3]), k, v, seen.expand(len(st["lens"]), n, nk))
    o = o.reshape(q.shape).transpose(1, 2)  # [B, n, Hq, D]
    real = torch.arange(n, device=DEV) < (st["cu"][1:] - st["cu"][:-1]).unsqueeze(1)
    out = torch.empty(st["q"].shape, device=DEV)
    at = (st["cu"][:-1].long().unsqueeze(1) + torch.arange(n, device=DEV))
    out.index_put_((torch.where(real, at, at[:, :1]),), torch.where(real.view(*real.shape, 1, 1), o, o[:, :1]))
    return {"o": out.to(st["q"].dtype)}


def _paged(st):
    case, table = st["case"], st["table"].long().clamp(min=0)
    b, hk, n = case["batch"], case["kv_heads"], case["max_len"]
    k, v = (st[x][table].float().transpose(1, 2).reshape(b, hk, -1, case["head_dim"])[:, :, :n]
            for x in ("k_pages", "v_pages"))
    j, lens = torch.arange(n, device=DEV), st["seqlens"].unsqueeze(1)
    seen = j < lens
    if case["window"] >= 0:
        seen = seen & (j >= lens - 1 - case["window"])
    o = _attend(st["q"].float().view(b, hk, -1, 1, case["head_dim"]), k, v, seen.unsqueeze(1))
    return {"o": o.reshape(st["q"].shape).to(st["q"].dtype)}


def _write(st):
    case = st["case"]
    hq, hk, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
    x = st["qkv"].view(n, hq + 2 * hk, d)
    cos, sin = (st[c][st["positions"].long()].float().unsqueeze(1) for c in ("cos", "sin"))

    def turned(y, w):
        y = y.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        half = torch.cat([-y[..., d // 2 :], y[..., : d // 2]], -1)
        return (y * cos + half * sin).to(x.dtype)

    q, k = turned(x[:, :hq], st["q_norm"]), turned(x[:, hq : hq + hk], st["k_norm"])
    page, row = st["slots"] // case["page"], st["slots"] % case["page"]
    st["k_pages"][page, :, row] = k
    st["v_pages"][page, :, row] = x[:, hq + hk :]
    return {"q": q, "k": k, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _logprobs(st):
    x, top = st["logits"].float(), st["case"]["top"]
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    z = e.sum(-1, keepdim=True)
    log_z = z.log()
    out = {"logprobs": (x.gather(1, st["tokens"].unsqueeze(1)) - log_z).squeeze(1),
           "entropy": (log_z - (e * x).sum(-1, keepdim=True) / z).squeeze(1)}
    if top:
        best, at = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_logprobs"], out["top_tokens"] = best[:, :top] - log_z, at[:, :top]
    return out


# ---- the calls a user makes --------------------------------------------------------


def _own(st):
    case, op = st["case"], st["case"]["op"]
    if op == "packed":
        from torchplusplus_amd.attention import packed_attention
        return {"o": packed_attention(st["q"], st["k"], st["v"], st["cu"], st["cu_k"] if case["prefix"] else None,
                                      causal=True, window_size=(case["window"], -1))}
    if op == "paged":
        from torchplusplus_amd.attention import paged_attention
        return {"o": paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seqlens"],
                                     window_left=case["window"])}
    if op == "write":
        from torchplusplus_amd.llmops.paged import qkv_rope_paged
        q, k = qkv_rope_paged(st["qkv"], st["positions"], st["slots"], st["k_pages"], st["v_pages"], st["cos"],
                              st["sin"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS)
        return {"q": q, "k": k, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    from torchplusplus_amd.llmops.scoring import token_logprobs
    r = token_logprobs(st["logits"], st["tokens"], top_k=case["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs, r.top_tokens
    return out


def run(state):
    if own:
        return _own(state)
    return {"packed": _packed, "paged": _paged, "write": _write, "logprobs": _logprobs}[state["case"]["op"]](state)


# ---- what a pass cannot do without, and its result in 64 bits -------------------------


def work(case):
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * (16 + 12 * case["top"]),
                "flops": 4 * n}
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if op == "packed":
        n = sum(_lengths(case))
        nk = n + case["prefix"] * case["batch"]
        if case["window"] >= 0:  # keys before the first query's window are never seen
            nk -= case["batch"] * max(0, case["prefix"] - case["window"])
        return {"bytes": 4 * n * hq * d + 4 * nk * hk * d, "flops": 4 * _pairs(case) * hq * d}
    if op == "paged":
        most = case["window"] + 1 if case["window"] >= 0 else case["max_len"]
        keys = sum(min(x, most) for x in _lengths(case))
        return {"bytes": 4 * keys * hk * d + 4 * case["batch"] * hq * d, "flops": 4 * keys * hq * d}
    n = case["tokens"]
    # read q, k, v; write q, k, and k and v in their pages
    return {"bytes": 2 * n * d * (2 * hq + 5 * hk) + 12 * n, "flops": 8 * n * (hq + hk) * d}


def exact(case, seed):
    op = case["op"]
    if op == "logprobs":
        if case["rows"] * case["vocab"] > 2e8:
            return None
        st = prepare(case, seed)
        out = {"logprobs": [], "entropy": []}
        if case["top"]:
            out["top_logprobs"] = []
        for r in range(case["rows"]):
            lp = torch.log_softmax(st["logits"][r].double(), 0)
            out["logprobs"].append(lp[st["tokens"][r]])
            out["entropy"].append(-(lp.exp() * lp).sum())
            if case["top"]:
                out["top_logprobs"].append(lp.topk(case["top"]).values)
        out = {n: torch.stack(x) for n, x in out.items()}
        if case["top"]:
            out["top_tokens"] = None
        return out
    st = prepare(case, seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    g = hq // hk
    if op == "write":
        x = st["qkv"].double().view(case["tokens"], -1, d)
        out = {}
        a, b = x[..., : d // 2], x[..., d // 2 :]
        c, s = (st[t].double()[st["positions"].long()][:, None, : d // 2] for t in ("cos", "sin"))
        for n, rows, w in (("q", slice(0, hq), st["q_norm"]), ("k", slice(hq, hq + hk), st["k_norm"])):
            lo, hi = a[:, rows], b[:, rows]
            if w is not None:
                r = ((lo * lo).sum(-1, keepdim=True) + (hi * hi).sum(-1, keepdim=True)) / d + EPS
                lo, hi = lo / r.sqrt() * w[: d // 2].double(), hi / r.sqrt() * w[d // 2 :].double()
            out[n] = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
        for n, rows in (("k_pages", out["k"]), ("v_pages", x[:, hq + hk :])):
            pages = st[n].double().transpose(1, 2).reshape(-1, hk, d)
            pages[st["slots"]] = rows
            out[n] = pages.view(-1, case["page"], hk, d).transpose(1, 2)
        return out
    o = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    if op == "packed":
        if _pairs(case) * hq * d > 2e12:
            return None
        a = b = 0
        for n in st["lens"]:
            nk = n + case["prefix"]
            i = torch.arange(n, device=DEV).unsqueeze(1) + case["prefix"]
            j = torch.arange(nk, device=DEV)
            hide = j > i
            if case["window"] >= 0:
                hide |= j < i - case["window"]
            for h in range(hq):
                s = st["q"][a : a + n, h].double() @ st["k"][b : b + nk, h // g].double().T / math.sqrt(d)
                s[hide] = -math.inf
                o[a : a + n, h] = torch.softmax(s, -1) @ st["v"][b : b + nk, h // g].double()
            a, b = a + n, b + nk
        return {"o": o}
    for i, n in enumerate(st["lens"]):
        lo = max(0, n - 1 - case["window"]) if case["window"] >= 0 else 0
        pages = st["table"][i, : -(-n // case["page"])].long()
        for h in range(hk):
            k, v = (st[x][pages, h].double().reshape(-1, d)[lo:n] for x in ("k_pages", "v_pages"))
            s = st["q"][i, h * g : (h + 1) * g].double() @ k.T / math.sqrt(d)
            o[i, h * g : (h + 1) * g] = torch.softmax(s, -1) @ v
    return {"o": o}
