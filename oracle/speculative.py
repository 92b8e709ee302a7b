"""Plain 64-bit forms of the speculative-decoding operators (CPU): rotation at
positions, cache codes, tree attention, verification."""
from __future__ import annotations

import math

import torch

CODE_MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
# the largest value below 2^128 that a row of codes holds
VALUE_MAX = {torch.float8_e4m3fn: 240 * 2.0 ** 120, torch.int8: 127 * 2.0 ** 121}


def rope_at(x, positions, inv_freq, interleaved=False, factor=1.0):
    """x [B, S, H, D], positions [B, S] or [S] -> fp64, and the size of the
    terms each element is made of (for its tolerance)."""
    x = x.double()
    out, terms = x.clone(), x.abs()
    half = len(inv_freq)
    pos = positions.long().expand(x.shape[0], x.shape[1]) if positions.dim() == 1 else positions.long()
    for b in range(x.shape[0]):
        for s in range(x.shape[1]):
            p = int(pos[b, s])
            if p < 0:
                continue
            for j in range(half):
                t = p * float(inv_freq[j])
                c, sn = math.cos(t) * factor, math.sin(t) * factor
                i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
                a, d = x[b, s, :, i], x[b, s, :, k]
                out[b, s, :, i], out[b, s, :, k] = a * c - d * sn, d * c + a * sn
                terms[b, s, :, i] = terms[b, s, :, k] = (a.abs() + d.abs()) * abs(factor)
    return out, terms


def quantise(x, code_dtype):
    """Rows [..., D] -> (code values fp64, exponent bytes)."""
    x, most = x.double(), CODE_MAX[code_dtype]
    rows = x.reshape(-1, x.shape[-1])
    codes, exps = torch.zeros_like(rows), torch.zeros(len(rows), dtype=torch.uint8)
    for i, r in enumerate(rows):
        if not bool(torch.isfinite(r).all()):
            exps[i] = 255
            continue
        r = r.clamp(-VALUE_MAX[code_dtype], VALUE_MAX[code_dtype])
        amax, e = float(r.abs().max()), -126
        while amax > most * 2.0 ** e:
            e += 1
        exps[i] = e + 127
        y = r * 2.0 ** -e
        if code_dtype == torch.int8:
            codes[i] = y.round()
        else:  # 3 bits after the first, 2^-9 the least step
            step = torch.tensor([2.0 ** (max(math.frexp(v)[1] - 1, -6) - 3) for v in y.tolist()],
                                dtype=torch.float64)
            codes[i] = (y / step).round() * step
    return codes.reshape(x.shape), exps.reshape(x.shape[:-1])


def values(codes, exps):
    """What codes [..., D] and exponent bytes [...] stand for, in fp64."""
    e = exps.double().unsqueeze(-1)
    v = codes.to(torch.float32).double() * torch.exp2(e - 127)
    return torch.where(e == 255, torch.full_like(v, math.nan), v)


def sees(parents, t):
    """The drafted tokens that token t sees (None: padding)."""
    out, at = [], t
    while at != -1:
        out.append(at)
        p = int(parents[at])
        if p < -1 or p >= at:
            return None
        at = p
    return out


def tree_attention(q, k, v, seqlens, parents=None, scale=None):
    """q [B, T, Hq, D], k, v [B, Hkv, L, D] values -> o in fp64, the weighted
    mean of |v| behind each element, and the largest sum of |q k| scale."""
    q, k, v = q.double(), k.double(), v.double()
    nb, nt, hq, d = q.shape
    hkv, room = k.shape[1], k.shape[2]
    scale = scale or 1.0 / math.sqrt(d)
    o, mean, size = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for b in range(nb):
        n = min(max(int(seqlens[b]), 0), room)
        for t in range(nt):
            own = sees(parents[b] if parents is not None else range(-1, nt - 1), t)
            if own is None or n + t >= room:
                continue
            keys = list(range(n)) + sorted(n + i for i in own)
            for h in range(hq):
                kk, vv = k[b, h // (hq // hkv), keys], v[b, h // (hq // hkv), keys]
                w = torch.softmax((kk @ q[b, t, h]) * scale, 0)
                o[b, t, h], mean[b, t, h] = w @ vv, w @ vv.abs()
                size = max(size, float((kk.abs() @ q[b, t, h].abs()).max()) * scale)
    return o, mean, size


def _mass(x):
    return float(x) if 0.0 < float(x) < math.inf else 0.0


def verify_draft(tokens, target, uniforms, draft=None, parents=None):
    """(accepted, path, next token), one sequence after the other."""
    nb, nt = tokens.shape
    accepted, path, nxt = [], torch.full((nb, nt), -1, dtype=torch.int32), []
    vocab = target.shape[2]

    def clean(row):
        row = row.double().clone()
        row[~((row > 0) & (row < math.inf))] = 0.0
        return row

    for b in range(nb):
        tok = [int(t) for t in tokens[b]]
        good = [0 <= t < vocab for t in tok]
        u = [float(x) for x in uniforms[b]]
        steps = []
        if draft is not None:
            n = 0
            while n < nt and good[n] and u[n] * _mass(draft[b, n, tok[n]]) < _mass(target[b, n, tok[n]]):
                steps.append(n)
                n += 1
            row = clean(target[b, n])
            rest = row.clone()
            if n < nt and good[n]:
                rest = (row - clean(draft[b, n])).clamp(min=0)
        else:
            par = [int(parents[b, i]) if parents is not None else i - 1 for i in range(nt)]
            node = -1
            while len(steps) < nt:
                below, seen, found = 0.0, set(), None
                for i in range(nt):
                    if par[i] != node or i <= node or not good[i] or tok[i] in seen:
                        continue
                    seen.add(tok[i])
                    m = _mass(target[b, node + 1, tok[i]])
                    if below <= u[len(steps)] < below + m:
                        found = i
                        break
                    below += m
                if found is None:
                    break
                steps.append(found)
                node = found
            row = clean(target[b, node + 1])
            rest = row.clone()
            for i in range(nt):
                if par[i] == node and i > node and good[i]:
                    rest[tok[i]] = 0.0
        accepted.append(len(steps))
        path[b, : len(steps)] = torch.tensor(steps, dtype=torch.int32)
        if float(rest.sum()) == 0.0:
            rest = row
        cum = rest.cumsum(0)
        hit = (cum > max(u[nt], 0.0) * cum[-1]).nonzero()
        left = rest.nonzero()
        nxt.append(-1 if not len(left) else int(hit[0]) if len(hit) else int(left[-1]))
    return torch.tensor(accepted, dtype=torch.int32), path, torch.tensor(nxt)
