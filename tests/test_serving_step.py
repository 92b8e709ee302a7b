"""The operators of a mixed batch together, as a serving program uses them, and the paths
of the framework that call them."""
import pytest
import torch

from oracle import serving as oracle
from oracle.qwen3 import Qwen3Oracle
from tests.conftest import close
from tests.test_model import TINY, TINY16, _oracle32, _rel
from tests.test_packed_attention import tolerance
from tests.test_rope_paged import tables


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_steps(dev, dtype, d):
    """Prompts of different lengths, decode steps, a sequence that ends and one that takes
    its pages, a follow-up turn: after each, attention of every new token must be that over
    a plain record of its sequence's rotated keys and values."""
    from torchplusplus_amd.attention import packed_attention, paged_attention
    from torchplusplus_amd.llmops.paged import PagedKVCache, qkv_rope_paged
    hq, hk, page = 8, 4, 16
    g = torch.Generator().manual_seed(5)
    cos, sin = tables(512, d, torch.float32, dev)
    cache = PagedKVCache(20, page, 1, hk, d, dtype, dev)
    kp, vp = cache.k_pages[0], cache.v_pages[0]
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(dtype).to(dev) for _ in "qk"]
    record = {}  # sequence: its keys and values, as the pages hold them

    def project(step):
        n = len(step.positions)
        qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(dtype).to(dev)
        q, k = qkv_rope_paged(qkv, step.positions, step.slots, kp, vp, cos, sin, *w)
        return q, k, qkv[:, (hq + hk) * d :].unflatten(1, (hk, d))

    def note(seqs, counts, k, v):
        at = 0
        for s, n in zip(seqs, counts):
            new = [x[at : at + n].cpu() for x in (k, v)]
            record[s] = [torch.cat(x) for x in zip(record[s], new)] if s in record else new
            at += n

    def check(got, seqs, counts, q):
        at = 0
        for s, n in zip(seqs, counts):
            k, v = record[s]
            o, mean, size = oracle.packed_attention(q[at : at + n], k, v, [0, n], [0, len(k)])
            tol = tolerance(o, mean, size, dtype, len(k), d, float(v.abs().max().float()))
            assert ((got[at : at + n].double().cpu() - o).abs() <= tol).all(), (s, n)
            at += n

    def prefill(seqs, starts, counts):
        step = cache.prefill_step(seqs, starts, counts)
        q, k, v = project(step)
        note(seqs, counts, k, v)
        if step.key_slots is not None:
            k, v = cache.read(0, step.key_slots)
        check(packed_attention(q, k, v, step.cu_seqlens, step.cu_seqlens_k), seqs, counts, q)

    def decode(seqs, steps):
        lens = [len(record[s][0]) for s in seqs]
        for s, n in zip(seqs, lens):
            cache.grow(s, n + steps)
        table, pos = cache.block_tables(seqs), torch.tensor(lens, dtype=torch.int32, device=dev)
        for _ in range(steps):
            step = cache.decode_step(table, pos)
            q, k, v = project(step)
            note(seqs, [1] * len(seqs), k, v)
            check(paged_attention(q, kp, vp, step.block_tables, step.seqlens), seqs, [1] * len(seqs), q)
            pos = pos + 1

    a, b, c = (cache.allocate() for _ in range(3))
    prefill([a, b, c], [0, 0, 0], [37, 1, 70])
    decode([a, b, c], 3)
    cache.free(b)
    e = cache.allocate()
    prefill([e], [0], [50])  # over b's page
    decode([c, e, a], 2)
    prefill([a, e], [len(record[a][0]), 0 + len(record[e][0])], [33, 9])
    decode([a, c], 15)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.prefill_step([a, c], [len(record[a][0]), len(record[c][0])], [100, 200])
    decode([e], 1)  # nothing was dealt


def model_close(got, exp, exp32, what):
    """The oracle rounds between the norm and the rotation of q and k, the paged path does
    not. Where two bf16 evaluations round in other places, each is off the fp32 one by an
    error of its own, e and e', and they are up to e + e' apart (the triangle inequality),
    so a bound on their distance that holds for one order of roundings says nothing about
    another. What is asked is that e' is no more than test_model.py asks of it: 1.25 e + 2e-3,
    the largest 1.5 times the oracle's largest + 5e-3. fp16: its tolerance."""
    if got.dtype == torch.float16:
        close(got, exp, what=what)
    e, orc = _rel(got, exp32), _rel(exp, exp32)
    assert e <= 1.25 * orc + 2e-3, f"{what}: error vs fp32 {e:.5f}, oracle's own {orc:.5f}"
    m, m_orc = ((x.float() - exp32.float()).abs().max().item() for x in (got, exp))
    assert m <= 1.5 * m_orc + 5e-3, f"{what}: max error vs fp32 {m:.4f}, oracle's own {m_orc:.4f}"


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [TINY, TINY16])
def test_model_paged_against_oracle(dev, cfg):
    """Packed prefill, decode and a follow-up turn of FastQwen3 over pages, each sequence
    against the oracle on its own."""
    from torchplusplus_amd.fastqwen3 import FastQwen3
    from torchplusplus_amd.llmops.paged import PagedKVCache
    with torch.inference_mode():
        m = FastQwen3(cfg, device=dev).eval()
        m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(1))
        g = torch.Generator().manual_seed(2)
        lens, turn = [40, 3, 129], [5, 30, 1]
        ids = [torch.randint(0, cfg.vocab_size, (n + 2 + t,), generator=g) for n, t in zip(lens, turn)]
        want, exact = [], []
        for x in ids:
            orc = Qwen3Oracle(m.state_dict(), cfg, cfg.context_length)
            exact.append(_oracle32(orc, cfg).forward(x.view(1, -1), 0)[0])
            want.append(orc.forward(x.view(1, -1), 0)[0])
        cache = PagedKVCache(24, 16, cfg.n_layers, cfg.n_kv_heads, cfg.head_dim, cfg.dtype, dev)
        seqs = [cache.allocate(n + 2) for n in lens]

        def packed(starts, counts):
            step = cache.prefill_step(seqs, starts, counts)
            toks = torch.cat([x[a : a + n] for x, a, n in zip(ids, starts, counts)]).to(dev)
            got = m.forward_paged(toks, cache, step).cpu()
            for i, x in enumerate(got.split(counts)):
                at = slice(starts[i], starts[i] + counts[i])
                model_close(x, want[i][at], exact[i][at], f"sequence {i} from {starts[i]}")
            return toks, step, got

        toks, step, got = packed([0, 0, 0], lens)
        last = m.forward_paged(toks, cache, step, step.cu_seqlens[1:].long() - 1).cpu()
        at = [n - 1 for n in lens]
        model_close(last, torch.stack([x[n] for x, n in zip(want, at)]), torch.stack([x[n] for x, n in zip(exact, at)]),
                    "last rows")
        pos = torch.tensor(lens, dtype=torch.int32, device=dev)
        for s in range(2):
            toks = torch.stack([x[n + s] for x, n in zip(ids, lens)]).to(dev)
            got = m.forward_paged(toks, cache, cache.decode_step(cache.block_tables(seqs), pos + s)).cpu()
            for i, n in enumerate(lens):
                model_close(got[i], want[i][n + s], exact[i][n + s], f"sequence {i}, token {n + s}")
        packed([n + 2 for n in lens], turn)


@pytest.mark.gpu
def test_generate_paged(dev):
    """Tokens are the largest logits' of a forward pass over what was generated, one
    sequence at a time (within the pass's own rounding), log probabilities that pass's."""
    from torchplusplus_amd.fastqwen3 import FastQwen3
    from torchplusplus_amd.llmops.scoring import token_logprobs
    cfg = TINY16
    with torch.inference_mode():
        m = FastQwen3(cfg, device=dev).eval()
        m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(3))
        g = torch.Generator().manual_seed(4)
        prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (7, 150, 1, 64)]
        toks, scores = m.generate_paged(prompts, 9, page_size=16, top_k=4)
        assert toks.shape == (4, 9) and scores.logprobs.shape == (4, 9) and scores.top_tokens.shape == (4, 9, 4)
        assert torch.equal(scores.top_tokens[..., 0], toks)
        for i, p in enumerate(prompts):
            seq = torch.cat([p.to(dev), toks[i]])
            logits = m.forward(seq.view(1, -1))[0, len(p) - 1 : -1].float()
            best = logits.amax(1)
            chosen = logits.gather(1, toks[i].unsqueeze(1)).squeeze(1)
            assert (best - chosen <= 0.05).all(), (i, best - chosen)
            ref = token_logprobs(logits, toks[i])
            assert (scores.logprobs[i] - ref.logprobs).abs().max() < 0.06
            assert (scores.entropy[i] - ref.entropy).abs().max() < 0.06
        same, none = m.generate_paged(prompts, 9, page_size=128)
        assert torch.equal(same, toks) and none.top_tokens is None
        for bad in (([], 3), ([prompts[0][:0]], 3), (prompts, 0), ([prompts[1]], cfg.context_length)):
            with pytest.raises(ValueError):
                m.generate_paged(*bad)


@pytest.mark.gpu
def test_score(dev):
    from torchplusplus_amd.fastqwen3 import FastQwen3
    cfg = TINY
    with torch.inference_mode():
        m = FastQwen3(cfg, device=dev).eval()
        m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(5))
        ids = torch.randint(0, cfg.vocab_size, (2, 33), generator=torch.Generator().manual_seed(6)).to(dev)
        got = m.score(ids, top_k=3)
        logits = m.forward(ids)
        for b in range(2):
            lp, ent, best, at = oracle.logprobs(logits[b, :-1], ids[b, 1:], 3)
            assert (got.logprobs[b].double().cpu() - lp).abs().max() < 1e-4
            assert (got.entropy[b].double().cpu() - ent).abs().max() < 1e-4
            assert (got.top_logprobs[b].double().cpu() - best).abs().max() < 1e-4
            assert torch.equal(got.top_tokens[b].cpu(), at)
        assert got.logprobs.shape == (2, 32) and m.score(ids).top_tokens is None
        for bad in (ids[0], ids[:, :1]):
            with pytest.raises(ValueError):
                m.score(bad)
