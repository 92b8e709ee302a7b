"""The speculative-decoding operators together, as a serving step uses them, and
the paths of the framework that call them."""
import pytest
import torch

from oracle import speculative as osp
from tests.test_tree_attention import CODES, check, tolerance, tree


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", CODES)
def test_steps(dev, dtype, code):
    """Three steps over a padded batch: rotate the drafted tokens at their
    depths, append, attend with the tree, verify, keep the accepted rows. After
    each the cache must hold the accepted sequence, row by row, and attention of
    the next tree must be that over a plain record of it."""
    from torchplusplus_amd.attention import tree_attention
    from torchplusplus_amd.dlops.rope import rope_apply_at, rope_frequencies
    from torchplusplus_amd.llmops.kvcache import KVCache, QuantKVCache
    from torchplusplus_amd.llmops.speculative import verify_draft
    b, t, hq, hkv, d, room, vocab = 3, 9, 8, 4, 64, 96, 50
    g = torch.Generator().manual_seed(3)
    freq, factor = rope_frequencies(d, 1e4, "yarn", 4.0, original_context=1024, device=dev)
    lens = [40, 7, 0]
    if code is None:
        cache = KVCache(room, hkv, d, dtype, dev, b)
    else:
        cache = QuantKVCache(room, hkv, d, dtype, dev, b, code_dtype=code)

    def values():
        if code is None:
            return [cache.k_cache.cpu(), cache.v_cache.cpu()]
        kc, vc, ke, ve = cache.rows(b)
        return [osp.values(c.cpu(), e.cpu()) for c, e in ((kc, ke), (vc, ve))]

    def write(k, v, at, counts=None):
        if code is None:
            for i in range(b):
                n = int(counts[i]) if counts is not None else k.shape[1]
                for c, x in ((cache.k_cache, k), (cache.v_cache, v)):
                    c[i, :, at[i] : at[i] + n] = x[i, :n].transpose(0, 1)
        else:
            cache.append(k, v, torch.tensor(at, dtype=torch.int32, device=dev),
                         None if counts is None else counts.to(dev))

    def heads(s):
        qkv = torch.randn(b, s, (hq + 2 * hkv) * d, generator=g).to(dtype).to(dev)
        return (x.unflatten(-1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], -1))

    # prompts of different lengths in one padded batch
    _, k, v = heads(40)
    _, k = rope_apply_at(k, k, torch.arange(40, device=dev), freq, attention_factor=factor)
    write(k, v, [0] * b, torch.tensor(lens, dtype=torch.int32))
    record = [[x[i, :, : lens[i]].clone() for i in range(b)] for x in values()]
    for step in range(3):
        par = tree(b, t, step)
        depth = torch.tensor([[len(osp.sees(par[i], j)) - 1 for j in range(t)] for i in range(b)])
        pos = (torch.tensor(lens).unsqueeze(1) + depth).int().to(dev)
        q, k, v = heads(t)
        q, k = rope_apply_at(q, k, pos, freq, attention_factor=factor)
        write(k, v, lens)
        start = torch.tensor(lens, dtype=torch.int32, device=dev)
        kw = {}
        if code is None:
            rows = (cache.k_cache, cache.v_cache)
        else:
            *rows, ke, ve = cache.rows(b)
            kw = dict(k_exps=ke, v_exps=ve)
        o = tree_attention(q, *rows, start, par.to(dev), **kw)
        now = values()
        for i in range(b):  # the context's rows are the record
            for x, r in zip(now, record):
                assert torch.equal(x[i, :, : lens[i]], r[i])
        check(q, rows, kw, now, start.cpu(), par, dtype, f"step {step}", got=o)
        probs = torch.softmax(torch.randn(b, t + 1, vocab, generator=g), -1)
        tok = torch.randint(0, vocab, (b, t), generator=g)
        u = torch.rand(b, t + 1, generator=g) * 0.05  # most first children stay
        n, path, nxt = verify_draft(tok.to(dev), probs.to(dev), u.to(dev), parents=par.to(dev))
        wn, wpath, wnext = osp.verify_draft(tok, probs, u, None, par)
        assert torch.equal(n.cpu(), wn) and torch.equal(path.cpu(), wpath) and torch.equal(nxt.cpu(), wnext)
        cache.keep(start, path)
        for i in range(b):
            at = [lens[i] + int(j) for j in wpath[i] if j >= 0]
            for r, x in zip(record, now):
                r[i] = torch.cat([r[i], x[i, :, at]], 1)
            lens[i] += int(wn[i])
    final = values()
    for i in range(b):
        for x, r in zip(final, record):
            assert torch.equal(x[i, :, : lens[i]], r[i])
    assert sum(lens) > 47, "nothing was accepted in three steps"


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES[1:])
@pytest.mark.parametrize("seq,past", [(1, 0), (1, 70), (5, 70), (64, 3), (100, 0), (80, 30)])
def test_grouped_query_layer_on_codes(dev, code, seq, past):
    """GroupedQueryAttention on a QuantKVCache against attention over the values
    that the cache then holds, for one token, a few, and a prompt."""
    from torchplusplus_amd.attention import GroupedQueryAttention, flash_attn_func
    from torchplusplus_amd.attention._common import norm_rope_qk
    from torchplusplus_amd.dlops.rope import compute_rope_params
    from torchplusplus_amd.llmops.kvcache import QuantKVCache
    b, hq, hkv, d, dim = 2, 4, 2, 64, 256
    torch.manual_seed(seq)
    layer = GroupedQueryAttention(dim, hq, hkv, d, dtype=torch.bfloat16, device=dev).eval()
    cos, sin = compute_rope_params(d, 1e4, 256, device=dev)
    cache = QuantKVCache(200, hkv, d, torch.bfloat16, dev, 3, code_dtype=code)  # room for more
    with torch.inference_mode():
        if past:
            layer(torch.randn(b, past, dim, device=dev).bfloat16(), cos, sin, cache, 0)
        qkv = torch.randn(b, seq, (hq + 2 * hkv) * d, device=dev).bfloat16()
        q, k, _ = (x.unflatten(-1, (-1, d)) for x in qkv.clone().split([hq * d, hkv * d, hkv * d], -1))
        q, k = norm_rope_qk(q, k, layer.q_norm, layer.k_norm, cos[past : past + seq], sin[past : past + seq])
        got = layer.attend(qkv, cos, sin, cache, past).view(b, seq, hq, d)
        assert cache.cache_len == past + seq and cache.batch_size == 3
        kc, vc, ke, ve = cache.rows(b)
        assert torch.equal(ke[:, :, past : past + seq].cpu(), osp.quantise(k.cpu(), code)[1].transpose(1, 2))
        vals = [osp.values(c.cpu(), e.cpu()) for c, e in ((kc, ke), (vc, ve))]
        if seq <= 64:
            o, mean, size = osp.tree_attention(q.cpu(), *vals, [past] * b)
            tol = tolerance(o, mean, size, torch.bfloat16, True, past + seq, d)
            assert bool(((got.double().cpu() - o).abs() <= tol).all())
        else:  # flash attention over the decoded prefix
            kk, vv = (x[:, :, : past + seq].bfloat16().to(dev).transpose(1, 2) for x in vals)
            assert torch.equal(got, flash_attn_func(q, kk, vv, causal=True))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES[1:])
def test_model_generates_over_codes(dev, code):
    """generate() over caches of codes: the caches keep their kind and are used,
    two runs agree; the captured decode refuses them, clear_kv_cache() goes back."""
    from tests.test_model import TINY
    from torchplusplus_amd.fastqwen3 import FastQwen3
    from torchplusplus_amd.llmops.kvcache import KVCache, QuantKVCache
    m = FastQwen3(TINY, device=dev).eval()
    m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(0))
    ids = torch.randint(0, TINY.vocab_size, (2, 30), generator=torch.Generator().manual_seed(1)).to(dev)
    m.setup_kv_cache(20, 2, code_dtype=code)
    out = m.generate(ids, max_new_token=8, sampling_strategy="greedy")
    assert all(isinstance(c, QuantKVCache) and c.code_dtype == code for c in m.kv_cache_array)
    assert out.shape == (2, 38) and m.kv_cache_array[0].cache_len == 37
    assert bool(m.kv_cache_array[-1].read(37)[1].abs().sum(-1).min() > 0), "rows were not written"
    assert torch.equal(out, m.generate(ids, max_new_token=8, sampling_strategy="greedy"))
    with pytest.raises(ValueError, match="16-bit"):
        m.generate_greedy(ids, 4)
    m.clear_kv_cache()
    assert m.generate_greedy(ids, 4).shape == (2, 34) and isinstance(m.kv_cache_array[0], KVCache)


@pytest.mark.gpu
def test_sample_draft(dev):
    """LLMInference.sample_draft is verify_draft on softmax(logits / temp)."""
    from tests.test_llmops import TinyLM
    g = torch.Generator().manual_seed(2)
    logits, tok = torch.randn(2, 4, 30, generator=g).to(dev), torch.randint(0, 30, (2, 3), generator=g)
    u = torch.rand(2, 4, generator=g)
    got = TinyLM().sample_draft(tok.to(dev), logits, 0.7, u.to(dev))
    want = osp.verify_draft(tok, torch.softmax(logits / 0.7, -1).cpu(), u)
    assert all(torch.equal(a.cpu(), w) for a, w in zip(got, want))
    n, path, nxt = TinyLM().sample_draft(tok.to(dev), logits.bfloat16())
    assert n.shape == (2,) and path.shape == (2, 3) and bool((nxt >= 0).all())


def test_setup_keeps_the_kind_of_cache():
    from tests.test_llmops import TinyLM
    from torchplusplus_amd.llmops.kvcache import KVCache, QuantKVCache

    class Wide(TinyLM):
        def get_head_dim(self):
            return 64

        def get_dtype(self):
            return torch.float16

    m = Wide()
    m.setup_kv_cache(16, 1)
    assert isinstance(m.kv_cache_array[0], KVCache)
    m.setup_kv_cache(16, 1, code_dtype=torch.int8)
    first = m.kv_cache_array
    assert isinstance(first[0], QuantKVCache)
    m.setup_kv_cache(8, 1)
    assert m.kv_cache_array is first
    m.setup_kv_cache(32, 2)
    assert isinstance(m.kv_cache_array[0], QuantKVCache) and m.kv_cache_array[0].code_dtype == torch.int8
    m.setup_kv_cache(32, 2, code_dtype=torch.float8_e4m3fn)
    assert m.kv_cache_array[0].code_dtype == torch.float8_e4m3fn
    m.kv_cache_array = None
    m.setup_kv_cache(32, 2)
    assert isinstance(m.kv_cache_array[0], KVCache)
