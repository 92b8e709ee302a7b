"""Plain 64-bit forms of the operators of a mixed batch over a paged cache (CPU):
packed and paged attention, the step between projection and attention, log
probabilities. Only what a row sees enters it."""
from __future__ import annotations

import math

import torch


def attend(q, k, v, seen, scale):
    """q [n, D], k and v [m, D], seen [n, m] -> o, the weights' mean of |v|, and of each
    row the largest sum of |q k| scale (for tolerances), all fp64."""
    q, k, v = q.double(), k.double(), v.double()
    o, mean = torch.zeros_like(q), torch.zeros_like(q)
    size = torch.zeros(len(q), 1, dtype=torch.float64)
    if k.shape[0] == 0:
        return o, mean, size
    if bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all()):
        s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        w = torch.where(seen.any(1, keepdim=True), w, torch.zeros_like(w))
        return w @ v, w @ v.abs(), ((q.abs() @ k.abs().T) * scale).masked_fill(~seen, 0).amax(1, keepdim=True)
    for i in range(len(q)):
        at = seen[i].nonzero().view(-1)
        if len(at):
            w = torch.softmax((k[at] @ q[i]) * scale, 0).unsqueeze(1)
            o[i], mean[i] = (w * v[at]).sum(0), (w * v[at].abs()).sum(0)
            size[i] = (k[at].abs() @ q[i].abs()).max() * scale
    return o, mean, size


def packed_attention(q, k, v, cu_q, cu_k, scale=None, causal=True, window=(-1, -1)):
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    n, hq, d = q.shape
    g = hq // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = [torch.zeros(n, hq, x, dtype=torch.float64) for x in (d, d, 1)]
    for b in range(len(cu_q) - 1):
        a, e = min(max(cu_q[b], 0), n), min(cu_q[b + 1], n)
        ka, ke = min(max(cu_k[b], 0), len(k)), min(cu_k[b + 1], len(k))
        if e <= a:
            continue
        ke = max(ke, ka)
        i = torch.arange(e - a).view(-1, 1) + (ke - ka) - (e - a)
        j = torch.arange(ke - ka).view(1, -1)
        right = 0 if causal else window[1]
        seen = torch.ones(e - a, ke - ka, dtype=torch.bool)
        if right >= 0:
            seen &= j <= i + right
        if window[0] >= 0:
            seen &= j >= i - window[0]
        for h in range(hq):
            for x, y in zip(out, attend(q[a:e, h], k[ka:ke, h // g], v[ka:ke, h // g], seen, scale)):
                x[a:e, h] = y
    return out


def paged_attention(q, k_pages, v_pages, tables, lens, scale=None, left=-1):
    q, k_pages, v_pages = q.cpu(), k_pages.cpu(), v_pages.cpu()
    b, hq, d = q.shape
    pages, hk, page, _ = k_pages.shape
    scale = d ** -0.5 if scale is None else scale
    out = [torch.zeros(b, hq, x, dtype=torch.float64) for x in (d, d, 1)]
    for i in range(b):
        n = min(max(int(lens[i]), 0), tables.shape[1] * page)
        at = [j for j in range(max(0, n - 1 - left) if left >= 0 else 0, n) if 0 <= int(tables[i, j // page]) < pages]
        pg, row = [int(tables[i, j // page]) for j in at], [j % page for j in at]
        for h in range(hq):
            k, v = (x[pg, h * hk // hq, row] for x in (k_pages, v_pages))
            seen = torch.ones(1, len(at), dtype=torch.bool)
            for x, y in zip(out, attend(q[i, h : h + 1], k, v, seen, scale)):
                x[i, h] = y[0]
    return out


def qkv_rope(qkv, positions, cos, sin, hq, hk, q_norm=None, k_norm=None, eps=1e-6):
    """q, k, v of [N, (Hq + 2 Hk) * D] in fp64, and the size of the terms of q and k."""
    n, d = qkv.shape[0], cos.shape[1]
    x = qkv.double().cpu().view(n, hq + 2 * hk, d)
    cos, sin, pos = cos.double().cpu(), sin.double().cpu(), positions.long().cpu()
    real = ((pos >= 0) & (pos < len(cos))).view(n, 1, 1)
    row = pos.clamp(0, len(cos) - 1)
    out, terms = [], []
    for y, w in ((x[:, :hq], q_norm), (x[:, hq : hq + hk], k_norm)):
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
        half = torch.cat([-y[..., d // 2 :], y[..., : d // 2]], -1)
        c, s = cos[row].unsqueeze(1), sin[row].unsqueeze(1)
        out.append(torch.where(real, y * c + half * s, torch.zeros_like(y)))
        terms.append(torch.where(real, (y * c).abs() + (half * s).abs(), torch.zeros_like(y)))
    return out[0], out[1], x[:, hq + hk :], terms[0], terms[1]


def logprobs(logits, tokens, top=0):
    """(logprobs, entropy, top logprobs, top tokens) in fp64."""
    x = logits.double().cpu()
    n, v = x.shape
    bad = ~torch.isfinite(x.amax(1)) | torch.isnan(x).any(1) | (x == math.inf).any(1)
    lp = torch.log_softmax(x, 1)
    lp[bad] = math.nan
    ent = -torch.where(lp == -math.inf, torch.zeros_like(lp), lp.exp() * lp).sum(1)
    t = tokens.cpu()
    inside = (t >= 0) & (t < v)
    got = lp.gather(1, t.clamp(0, v - 1).unsqueeze(1)).squeeze(1)
    got = torch.where(inside, got, torch.zeros_like(got))
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    best = lp.gather(1, ids)
    ids[torch.isnan(x).any(1) | (x == math.inf).any(1)] = -1
    return got, ent, best, ids
