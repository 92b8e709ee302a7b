"""tree_attention against the 64-bit form in oracle/speculative.py.

Tolerance of an element o = sum w v: with A = sum w |v| (the oracle's second
result), its own rounding eps / 2 |o| (half the least fp16 step, 2^-25), the
rounding of the weights, u = 2^-9 in bfloat16 and 2^-12 in fp16 of each (coded
caches: bfloat16 always; fp16 weights below 2^-39 are cut to nothing, n 2^-39 A
in all), and fp32 arithmetic: a score's error is at most (D + 8) 2^-24 of
sum |q k| scale (the oracle's third result, which bounds |score| too) plus
2^-22, twice that as relative error of a weight and again of their sum, and sums
over n keys n 2^-24 A."""
import pytest
import torch

from oracle import speculative as osp

CODES = [None, torch.float8_e4m3fn, torch.int8]


def tolerance(o, mean, size, dtype, coded, n, d):
    eps = torch.finfo(dtype).eps
    u = 2.0 ** -9 if coded or dtype == torch.bfloat16 else 2.0 ** -12
    fp32 = 4 * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -22) + 2 * n * 2.0 ** -24
    return eps / 2 * o.abs() * (1 + eps) + 2.0 ** -25 + (2 * u + n * 2.0 ** -39 + fp32) * mean


def make(b, t, hq, hkv, d, room, dtype, code, seed, dev):
    """q and a cache of random rows; the values that the cache stands for."""
    from torchplusplus_amd.llmops.kvcache import kv_quant_append, kv_quant_read
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, t, hq, d, generator=g).to(dtype).to(dev)
    kv = [torch.randn(b, room, hkv, d, generator=g) * torch.exp(torch.randn(b, room, hkv, 1, generator=g) * 0.5)
          for _ in "kv"]
    kv = [x.to(dtype).to(dev) for x in kv]
    if code is None:
        kv = [x.transpose(1, 2).contiguous() for x in kv]
        return q, kv, {}, [x.cpu() for x in kv]
    codes = [torch.zeros(b, hkv, room, d, dtype=torch.uint8, device=dev).view(code) for _ in "kv"]
    exps = [torch.full((b, hkv, room), 127, dtype=torch.uint8, device=dev) for _ in "kv"]
    kv_quant_append(*kv, *codes, *exps, 0)
    return (q, codes, dict(k_exps=exps[0], v_exps=exps[1]),
            [osp.values(c.cpu(), e.cpu()) for c, e in zip(codes, exps)])


def tree(b, t, seed):
    g = torch.Generator().manual_seed(seed)
    p = [[int(torch.randint(max(-1, i - 6), i, (1,), generator=g)) for i in range(t)] for _ in range(b)]
    return torch.tensor(p, dtype=torch.int32)


def check(q, cache, kw, vals, lens, parents, dtype, what, scale=None, got=None):
    from torchplusplus_amd.attention import tree_attention
    dev = q.device
    if got is None:
        got = tree_attention(q, *cache, lens.to(dev), None if parents is None else parents.to(dev),
                             softmax_scale=scale, **kw)
    o, mean, size = osp.tree_attention(q.cpu(), *vals, lens, parents, scale)
    n = int(lens.max()) + q.shape[1]
    tol = tolerance(o, mean, size, dtype, bool(kw), n, q.shape[3])
    off = (got.double().cpu() - o).abs() - tol
    assert not bool((off > 0).any()) and not bool(torch.isnan(off).any()), \
        f"{what}: {int((~(off <= 0)).sum())} off, by up to {float(off.max())} more than allowed"
    return got


# B, T, Hq, Hkv, D, room, lengths: one token, no context, tile edges (32 and 64
# keys, one past), groups of 1, 2, 3, 8, more rows than a 32- and a 64-row tile,
# 64 tokens, pair counts that are a multiple of 8 and not, mixed lengths
SHAPES = [(1, 1, 2, 1, 128, 16, [0]), (1, 1, 1, 1, 64, 32, [31]), (2, 1, 16, 8, 128, 208, [77, 130]),
          (1, 5, 6, 2, 64, 96, [64]), (3, 16, 4, 4, 128, 160, [0, 33, 144]), (1, 33, 8, 1, 128, 128, [95]),
          (1, 64, 3, 1, 64, 80, [16]), (2, 7, 8, 4, 64, 1040, [1000, 517]), (1, 64, 16, 2, 128, 400, [300]),
          (4, 3, 2, 2, 64, 64, [61, 1, 32, 63 - 3]), (1, 9, 8, 8, 128, 2064, [2047])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_attention(dev, dtype, code, shape):
    b, t, hq, hkv, d, room, lens = shape
    q, cache, kw, vals = make(b, t, hq, hkv, d, room, dtype, code, 1 + t, dev)
    got = check(q, cache, kw, vals, torch.tensor(lens, dtype=torch.int32), tree(b, t, t), dtype, f"tree {shape}")
    again = check(q, cache, kw, vals, torch.tensor(lens, dtype=torch.int32), tree(b, t, t), dtype, "again")
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [16, 80, 96, 256])
def test_other_head_sizes(dev, code, d):
    """Head sizes without a matrix-core kernel; codes of 64, 128, 256 only come
    from the cache, others are written here directly."""
    b, t, hq, hkv, room = 2, 5, 4, 2, 48
    g = torch.Generator().manual_seed(d)
    q = torch.randn(b, t, hq, d, generator=g).bfloat16().to(dev)
    lens, par = torch.tensor([20, 43], dtype=torch.int32), tree(b, t, 3)
    if code is None:
        cache = [torch.randn(b, hkv, room, d, generator=g).bfloat16().to(dev) for _ in "kv"]
        vals, kw = [x.cpu() for x in cache], {}
    else:
        both = [osp.quantise(torch.randn(b, hkv, room, d, generator=g), code) for _ in "kv"]
        cache = [c.float().to(code).to(dev) for c, _ in both]
        kw = dict(k_exps=both[0][1].to(dev), v_exps=both[1][1].to(dev))
        vals = [osp.values(c, e) for c, e in both]
    check(q, cache, kw, vals, lens, par, torch.bfloat16, f"D {d}")


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [64, 128])
def test_chain_padding_and_the_caches_end(dev, code, d):
    """No parents: a chain. Padding and its children see nothing, tokens past
    the cache's end neither, lengths below 0 count as 0; a scale of one's own,
    an output with strides."""
    from torchplusplus_amd.attention import tree_attention
    b, t, hq, hkv, room = 4, 6, 4, 2, 64
    q, cache, kw, vals = make(b, t, hq, hkv, d, room, torch.bfloat16, code, 9, dev)
    lens = torch.tensor([0, 40, 61, 64], dtype=torch.int32)
    got = check(q, cache, kw, vals, lens, None, torch.bfloat16, "chain", scale=0.3)
    assert bool((got[2, 3:] == 0).all()) and bool((got[3] == 0).all()) and bool((got[2, :3] != 0).any())
    par = torch.tensor([[-1, -2, 1, 0, 99, 4], [2, -1, -1, 3, 1, 0], [-1, 0, 1, 1, 1, 1], [-1] * 6], dtype=torch.int32)
    lens = torch.tensor([5, 0, 30, -7], dtype=torch.int32)
    out = torch.full((b, t, 2 * hq, d), 5.0, dtype=torch.bfloat16, device=dev)
    o = tree_attention(q, *cache, lens.to(dev), par.to(dev), out=out[:, :, ::2], **kw)
    check(q, cache, kw, vals, lens, par, torch.bfloat16, "padding", got=o)
    assert bool((o[0, [1, 2, 4, 5]] == 0).all()) and bool((o[1, [0, 3, 5]] == 0).all())
    assert bool((out[:, :, 1::2] == 5.0).all()), "values beside the output were written"


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("d", [64, 128])
def test_non_finite_rows_reach_who_sees_them(dev, code, bad, d):
    """A drafted token's NaN or infinite row makes non-finite those that see it
    and nobody else; rows behind the last token never count."""
    from torchplusplus_amd.attention import tree_attention
    from torchplusplus_amd.llmops.kvcache import kv_quant_append
    b, t, hq, hkv, room, n = 1, 8, 4, 2, 96, 50
    q, cache, kw, vals = make(b, t, hq, hkv, d, room, torch.bfloat16, code, 4, dev)
    par = torch.tensor([[-1, -1, 0, 1, 2, 3, 0, 6]], dtype=torch.int32)
    lens = torch.tensor([n], dtype=torch.int32)
    full = lambda x: torch.full((1, 1, hkv, d), x, dtype=torch.bfloat16)  # noqa: E731
    for which in (0, 1):
        c = [x.view(torch.uint8).clone().view(x.dtype) for x in cache]
        e = {k: v.clone() for k, v in kw.items()}
        for j, r in ((n + 1, full(bad)), (n + t, full(bad)), (room - 1, full(float("nan")))):
            if code is None:
                c[which][:, :, j] = r[:, 0].to(dev)
            else:
                x = [torch.zeros_like(r).to(dev)] * 2
                x[which] = r.to(dev)
                keep = [y[:, :, j].clone() for y in (c[1 - which].view(torch.uint8), list(e.values())[1 - which])]
                kv_quant_append(*x, *c, e["k_exps"], e["v_exps"], j)
                c[1 - which].view(torch.uint8)[:, :, j], list(e.values())[1 - which][:, :, j] = keep
        o = tree_attention(q, *c, lens.to(dev), par.to(dev), **e)
        seen = [1, 3, 5]                      # token 1 and what descends from it
        rest = [i for i in range(t) if i not in seen]
        assert not bool(torch.isfinite(o[0, seen]).all(-1).any()), "a seen row left no trace"
        want = tree_attention(q, *cache, lens.to(dev), par.to(dev), **kw)
        eps = torch.finfo(torch.bfloat16).eps
        # the same numbers, perhaps by another order of sums: two roundings apart at most
        ok = (o[0, rest].float() - want[0, rest].float()).abs() <= eps * want[0, rest].float().abs() + 2 * eps
        assert bool(ok.all()), "a row that is not seen had an effect"


@pytest.mark.gpu
def test_strides_and_a_larger_batch(dev):
    """Queries out of a fused projection, a cache with room for more sequences
    and heads interleaved with positions, equal to the contiguous call."""
    from torchplusplus_amd.attention import tree_attention
    b, t, hq, hkv, d, room = 2, 4, 8, 4, 128, 80
    q, (k, v), _, vals = make(b, t, hq, hkv, d, room, torch.float16, None, 6, dev)
    lens, par = torch.tensor([70, 13], dtype=torch.int32, device=dev), tree(b, t, 2).to(dev)
    want = tree_attention(q, k, v, lens, par)
    big = torch.randn(b, t, (hq + 3) * d, device=dev).half()
    qv = big[..., d : d + hq * d].view(b, t, hq, d)
    qv.copy_(q)
    both = torch.randn(b + 1, room, hkv, 2 * d, device=dev).half()
    kv, vv = both[:b, ..., :d].transpose(1, 2), both[:b, ..., d:].transpose(1, 2)
    kv.copy_(k)
    vv.copy_(v)
    assert torch.equal(tree_attention(qv, kv, vv, lens, par), want)
    # unaligned rows
    flat = torch.zeros(q.numel() + 1, dtype=torch.float16, device=dev)
    qu = flat[1:].view(b, t, hq, d)
    qu.copy_(q)
    check(qu, (k, v), {}, vals, lens.cpu(), par.cpu(), torch.float16, "unaligned")


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_captured_two_graphs_and_two_streams(dev, code):
    """Two graphs captured before either is replayed, replays between eager
    calls, lengths advanced between replays; calls on two streams."""
    from torchplusplus_amd.attention import tree_attention
    d, room = 128, 1040
    q, cache, kw, _ = make(2, 5, 8, 4, d, room, torch.bfloat16, code, 8, dev)
    par, lens = tree(2, 5, 1).to(dev), torch.tensor([1000, 600], dtype=torch.int32, device=dev)
    q1 = q[:, :1].contiguous()
    tree_attention(q, *cache, lens, par, **kw)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = tree_attention(q, *cache, lens, par, **kw)
    with torch.cuda.graph(g2):
        o2 = tree_attention(q1, *cache, lens, None, **kw)
    for i in range(4):
        lens.sub_(90 * i)
        g1.replay()
        g2.replay()
        assert torch.equal(o1, tree_attention(q, *cache, lens, par, **kw))
        assert torch.equal(o2, tree_attention(q1, *cache, lens, None, **kw))
    want, want1 = (tree_attention(x, *cache, lens, None, **kw) for x in (q, q1))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            outs.append((tree_attention(q, *cache, lens, None, **kw), want))
        with torch.cuda.stream(s2):
            outs.append((tree_attention(q1, *cache, lens, None, **kw), want1))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)


@pytest.mark.gpu
def test_many_calls_on_two_streams(dev):
    """Calls whose splits one launch merges, many times on two streams at once."""
    from torchplusplus_amd.attention import tree_attention
    b, hkv, d, room = 32, 8, 64, 1024
    q, cache, kw, _ = make(b, 1, 8, hkv, d, room, torch.bfloat16, torch.int8, 3, dev)
    lens = torch.randint(1, room - 1, (b,), generator=torch.Generator().manual_seed(1)).int()
    a, c = lens.to(dev), lens.flip(0).contiguous().to(dev)
    want = [tree_attention(q, *cache, x, None, **kw) for x in (a, c)]
    check(q, cache, kw, [osp.values(t.cpu(), e.cpu()) for t, e in zip(cache, (kw["k_exps"], kw["v_exps"]))], lens,
          None, torch.bfloat16, "mixed lengths", got=want[0])
    torch.cuda.synchronize()
    streams, bad = [torch.cuda.Stream() for _ in "ac"], []
    for s, x, w in zip(streams, (a, c), want):
        with torch.cuda.stream(s):
            bad.append(torch.zeros((), dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    for _ in range(700):
        for i, (s, x, w) in enumerate(zip(streams, (a, c), want)):
            with torch.cuda.stream(s):
                bad[i] += (tree_attention(q, *cache, x, None, **kw) != w).any()
    torch.cuda.synchronize()
    assert [int(n) for n in bad] == [0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("code", [None, torch.int8])
def test_offsets_past_32_bits(dev, code):
    """A cache whose last sequence begins past 2^32 bytes."""
    from torchplusplus_amd.attention import tree_attention
    b, hkv, d, room = 3, 8, 128, 1 << (20 if code is None else 21)
    dtype = torch.bfloat16 if code is None else code
    k = torch.zeros(b, hkv, room, d, dtype=dtype, device=dev)
    assert (b - 1) * hkv * room * d * k.element_size() >= 1 << 32
    kw = {}
    if code is not None:
        e = torch.full((b, hkv, room), 127, dtype=torch.uint8, device=dev)
        kw = dict(k_exps=e, v_exps=e)
    # keys 0, values 1 at the first and 3 at the last two positions: a mean
    k[:, :, 0], k[:, :, room - 2 :] = 1, 3
    q = torch.zeros(b, 1, 16, d, dtype=torch.bfloat16, device=dev)
    lens = torch.tensor([room - 1, 1, room - 1], dtype=torch.int32, device=dev)
    o = tree_attention(q, k, k, lens, None, **kw).float().cpu()
    want = torch.tensor([7.0 / room, 1.0 / 2, 7.0 / room])
    assert torch.allclose(o, want.view(b, 1, 1, 1).expand_as(o), rtol=2.0 ** -7)


def test_refuses_cpu_tensors():
    from torchplusplus_amd.attention import tree_attention
    q, c = torch.zeros(1, 1, 2, 64, dtype=torch.float16), torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        tree_attention(q, c, c, torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals(dev):
    from torchplusplus_amd.attention import tree_attention
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device=dev)
    c = torch.zeros(2, 2, 32, 64, dtype=torch.float16, device=dev)
    n, par = torch.zeros(2, dtype=torch.int32, device=dev), torch.full((2, 3), -1, dtype=torch.int32, device=dev)
    i8, e = c.to(torch.int8), torch.full((2, 2, 32), 127, dtype=torch.uint8, device=dev)
    ex = dict(k_exps=e, v_exps=e)
    for args, kw in (((q, c.bfloat16(), c, n), {}), ((q, c, c.bfloat16(), n), {}), ((q, c, c[:, :1], n), {}),
                     ((q, c[:1], c[:1], n), {}), ((q[:, :, :3], c, c, n), {}), ((q, c, c, n.long()), {}),
                     ((q, c, c, n[:1]), {}), ((q, c, c, n, par.long()), {}), ((q, c, c, n, par[:, :2]), {}),
                     ((q, c, c, n, par[:, :2].t()), {}), ((q, i8, i8, n), {}), ((q, c, c, n), ex),
                     ((q, i8, i8, n), dict(k_exps=e, v_exps=e[:, :, :16])), ((q, c, c, n.cpu()), {}),
                     ((q, i8, i8, n), dict(k_exps=e.int(), v_exps=e.int())), ((q.float(), c, c, n), {}),
                     ((q, c, c, n), dict(out=q[:, :2])), ((q[0], c, c, n), {}),
                     ((torch.zeros(2, 65, 4, 64, dtype=torch.float16, device=dev), c, c, n), {}),
                     ((torch.zeros(2, 1, 4, 512, dtype=torch.float16, device=dev),
                       torch.zeros(2, 2, 8, 512, dtype=torch.float16, device=dev),
                       torch.zeros(2, 2, 8, 512, dtype=torch.float16, device=dev), n), {})):
        with pytest.raises((RuntimeError, TypeError)):
            tree_attention(*args, **kw)
    assert tree_attention(q[:0], c[:0], c[:0], n[:0]).shape == (0, 3, 4, 64)


@pytest.mark.gpu
def test_stream_that_lags(dev):
    """A call that waits behind other work on its stream while another stream makes
    thousands: their blocks count themselves in on words of their own."""
    from torchplusplus_amd.attention import tree_attention
    q, cache, kw, _ = make(32, 1, 8, 8, 64, 1024, torch.bfloat16, torch.int8, 4, dev)
    lens = torch.randint(300, 1023, (32,), generator=torch.Generator().manual_seed(2)).int().to(dev)
    want = tree_attention(q, *cache, lens, None, **kw)
    busy = torch.randn(4096, 4096, device=dev)
    slow, fast, got = torch.cuda.Stream(), torch.cuda.Stream(), []
    torch.cuda.synchronize()
    with torch.cuda.stream(slow):
        for _ in range(20):
            busy @ busy
            got.append(tree_attention(q, *cache, lens, None, **kw))
    with torch.cuda.stream(fast):
        wrong = torch.zeros((), dtype=torch.int32, device=dev)
        for _ in range(1500):
            wrong += (tree_attention(q, *cache, lens, None, **kw) != want).any()
    torch.cuda.synchronize()
    assert int(wrong) == 0 and all(torch.equal(x, want) for x in got)


@pytest.mark.gpu
def test_refuses_an_out_that_is_not_its_own(dev):
    from torchplusplus_amd.attention import tree_attention
    q = torch.zeros(2, 3, 4, 64, dtype=torch.float16, device=dev)
    c = torch.zeros(2, 4, 3, 64, dtype=torch.float16, device=dev)
    n = torch.zeros(2, dtype=torch.int32, device=dev)
    for out in (q, c.view(2, 3, 4, 64), q[:1].expand(2, 3, 4, 64), torch.zeros_like(q)[:, :1].expand(2, 3, 4, 64)):
        with pytest.raises(RuntimeError, match="of its own"):
            tree_attention(q, c, c.clone(), n, out=out)
    both = torch.zeros(4, 3, 4, 64, dtype=torch.float16, device=dev)  # one buffer, two halves
    assert tree_attention(both[:2], c, c, n, out=both[2:]).data_ptr() == both[2:].data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("t,step", [(1, 0.05), (1, 0.4), (24, 0.05), (24, 0.4), (6, -0.05)])
def test_scores_that_rise_or_fall_along_the_keys(dev, dtype, code, t, step):
    """Scores that pass the running reference maximum by less and by more than its
    step of 2^8 from tile to tile, within a wave's tiles and between splits."""
    from torchplusplus_amd.llmops.kvcache import kv_quant_append
    b, hq, hkv, d, room, n = 2, 8, 4, 128, 1024, 900
    g = torch.Generator().manual_seed(t)
    q = torch.full((b, t, hq, d), 1.0)
    at = torch.arange(room, dtype=torch.float64).view(1, room, 1, 1)
    k = (at * step / d ** 0.5 + torch.randn(b, room, hkv, d, generator=g) * 0.02).to(dtype)
    v = torch.randn(b, room, hkv, d, generator=g).to(dtype)
    q, k, v = q.to(dtype).to(dev), k.to(dev), v.to(dev)
    if code is None:
        cache, kw = [x.transpose(1, 2).contiguous() for x in (k, v)], {}
        vals = [x.cpu() for x in cache]
    else:
        cache = [torch.zeros(b, hkv, room, d, dtype=torch.uint8, device=dev).view(code) for _ in "kv"]
        exps = [torch.full((b, hkv, room), 127, dtype=torch.uint8, device=dev) for _ in "kv"]
        kv_quant_append(k, v, *cache, *exps, 0)
        kw = dict(k_exps=exps[0], v_exps=exps[1])
        vals = [osp.values(c.cpu(), e.cpu()) for c, e in zip(cache, exps)]
    check(q, cache, kw, vals, torch.tensor([n, 37], dtype=torch.int32), None, dtype, (code, t, step))


@pytest.mark.gpu
def test_thousands_of_heads_of_one_kv_head(dev):
    """64 x 20000 query rows of one KV head: row / G by a multiplication in 32 bits
    would be off by one (row * G passes 2^32)."""
    from torchplusplus_amd.attention import tree_attention
    t, hq, d, room = 64, 20000, 64, 128
    q, cache, kw, vals = make(1, t, 16, 1, d, room, torch.float16, None, 6, dev)
    lens, parents = torch.tensor([5], dtype=torch.int32), tree(1, t, 2)
    many = torch.zeros(1, t, hq, d, dtype=torch.float16, device=dev)
    many[:, :, :8], many[:, :, -8:] = q[:, :, :8], q[:, :, 8:]
    got = tree_attention(many, *cache, lens.to(dev), parents.to(dev), **kw)
    got = torch.cat((got[:, :, :8], got[:, :, -8:]), 2)
    check(q, cache, kw, vals, lens, parents, torch.float16, "first and last heads", got=got)
