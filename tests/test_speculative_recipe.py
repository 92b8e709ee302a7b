"""A speculative decoding loop as the documentation gives it: the token drawn last is
the root of the next tree, so that its row is written with the drafted tokens'."""
import math

import pytest
import torch

from oracle import speculative as osp
from tests.test_tree_attention import CODES

B, HQ, HKV, D, VOCAB, ROOM = 3, 4, 2, 64, 50, 96


class Toy:
    """One attention layer between tables: a token's q, k and v are rows of them, the
    logits a product with the attention's output."""

    def __init__(self, dtype, dev):
        from torchplusplus_amd.dlops.rope import rope_frequencies
        g = torch.Generator().manual_seed(1)
        self.table = (1.5 * torch.randn(VOCAB, (HQ + 2 * HKV) * D, generator=g)).to(dtype)
        self.out = torch.randn(HQ * D, VOCAB, generator=g) / math.sqrt(HQ * D)
        self.freq, _ = rope_frequencies(D, 1e4, device="cpu")
        self.dtype, self.dev = dtype, dev

    def rows(self, tokens, positions):
        """Rotated q and k, and v, on the device, of tokens at positions [B, S]."""
        from torchplusplus_amd.dlops.rope import rope_apply_at
        x = self.table[tokens].to(self.dev)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split([HQ * D, HKV * D, HKV * D], -1))
        return (*rope_apply_at(q, k, positions.to(self.dev), self.freq.to(self.dev)), v)

    def logits(self, o):
        return o.flatten(2).float().cpu() @ self.out


def cache_of(code, dtype, dev):
    from torchplusplus_amd.llmops.kvcache import KVCache, QuantKVCache
    if code is None:
        return KVCache(ROOM, HKV, D, dtype, dev, B)
    return QuantKVCache(ROOM, HKV, D, dtype, dev, B, code_dtype=code)


def write(cache, k, v, at, counts=None):
    if hasattr(cache, "append"):
        cache.append(k, v, at, counts)
    else:
        for i in range(B):
            n = k.shape[1] if counts is None else int(counts[i])
            for c, x in ((cache.k_cache, k), (cache.v_cache, v)):
                c[i, :, int(at[i]) : int(at[i]) + n] = x[i, :n].transpose(0, 1)


def parts(cache):
    """The cache's tensors, and the exponents' arguments of tree_attention."""
    if hasattr(cache, "append"):
        kc, vc, ke, ve = cache.rows(B)
        return (kc, vc), dict(k_exps=ke, v_exps=ve)
    return (cache.k_cache, cache.v_cache), {}


def values(cache):
    c, e = parts(cache)
    return [x.cpu().double() for x in c] if not e else [osp.values(x.cpu(), y.cpu()) for x, y in zip(c, e.values())]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", CODES)
def test_loop_with_the_drawn_token_as_root(dev, dtype, code):
    """Greedy, over a padded batch of uneven lengths: after each step the cache holds the
    rows of the sequence so far, all but the token drawn last, as one append of that
    sequence would have left them, and every new token has the largest logit (within
    2%: one rounding of the attention's output and fp32 sums) of the 64-bit form."""
    from torchplusplus_amd.attention import tree_attention
    from tests.test_llmops import TinyLM
    toy, cache, t = Toy(dtype, dev), cache_of(code, dtype, dev), 8
    g = torch.Generator().manual_seed(2)
    seqs = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (30, 1, 12)]

    def reference(seq):
        """A cache with all of seq but its last token, and the logits behind that."""
        one = cache_of(code, dtype, dev)
        tok = torch.tensor([seq] * B)
        q, k, v = toy.rows(tok, torch.arange(len(seq)).int())
        write(one, k, v, torch.zeros(B, dtype=torch.int32, device=dev))
        vals = values(one)
        o, _, _ = osp.tree_attention(q[:1, -1:].cpu(), *[x[:1] for x in vals], [len(seq) - 1])
        return vals, toy.logits(o)[0, 0]

    # the prompts but for their last tokens, which are the first roots
    most = max(len(s) for s in seqs) - 1
    tok = torch.tensor([s[:-1] + [0] * (most - len(s) + 1) for s in seqs])
    lens = torch.tensor([len(s) - 1 for s in seqs], dtype=torch.int32, device=dev)
    _, k, v = toy.rows(tok, torch.arange(most).int())
    write(cache, k, v, torch.zeros(B, dtype=torch.int32, device=dev), lens)
    taken = 0
    for step in range(4):
        # a draft: the continuation, now and then wrong, among other children; padding
        draft, par = [], []
        for s in seqs:
            d, p, last, grown = [], [], -1, list(s)
            while len(d) < t:
                if torch.rand((), generator=g) < 0.4:
                    d.append(int(torch.randint(0, VOCAB, (), generator=g)))
                    p.append(last)
                else:
                    best = int(reference(grown)[1].argmax())
                    grown.append(best if torch.rand((), generator=g) < 0.9 else 7)
                    d.append(grown[-1])
                    p.append(last)
                    last = len(d) - 1
            p[-1] = -2
            draft.append(d)
            par.append(p)
        draft, par = torch.tensor(draft), torch.tensor(par, dtype=torch.int32)

        # 1. the last drawn token is node 0, the drafted tokens hang below it
        nodes = torch.cat([torch.tensor([[s[-1]] for s in seqs]), draft], 1)
        valid = (par >= -1) & (par < torch.arange(t))
        tree = torch.cat([torch.full((B, 1), -1), torch.where(valid, par + 1, -2)], 1).int()
        depth = torch.zeros(B, t + 1, dtype=torch.int32)
        for i in range(1, t + 1):
            depth[:, i] = depth.gather(1, tree[:, i : i + 1].clamp(min=0).long())[:, 0] + 1
        # 2. rotate at context + depth, append behind the context, attend
        q, k, v = toy.rows(nodes, lens.cpu().unsqueeze(1) + depth)
        write(cache, k, v, lens)
        c, e = parts(cache)
        logits = toy.logits(tree_attention(q, *c, lens, tree.to(dev), **e))
        # 3. verify: row 0 is the root's, row t + 1 drafted token t's
        n, path, nxt = TinyLM().sample_draft(draft.to(dev), logits.to(dev), 0.0, parents=par.to(dev))
        # 4. the accepted rows move behind the root's
        cache.keep(lens + 1, path)
        lens = lens + n + 1
        taken += int(n.sum())
        for i, s in enumerate(seqs):
            for x in [int(draft[i, j]) for j in path[i] if j >= 0] + [int(nxt[i])]:
                want = reference(s)[1]
                assert float(want.max() - want[x]) <= 0.02 * float(want.std()), f"step {step}, sequence {i}"
                s.append(x)
        now = values(cache)
        for i, s in enumerate(seqs):
            assert int(lens[i]) == len(s) - 1
            for x, r in zip(now, reference(s)[0]):
                assert torch.equal(x[i, :, : lens[i]], r[0, :, : lens[i]]), f"step {step}, sequence {i}"
    assert taken >= 6, "hardly anything was accepted"
