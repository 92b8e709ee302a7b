"""The cache of 8-bit codes against the 64-bit form in oracle/speculative.py:
codes, exponents and decoded bfloat16 values are equal bit by bit (powers of
two: nothing but the one rounding of an element)."""
import pytest
import torch

from oracle import speculative as osp
from torchplusplus_amd.llmops.kvcache import QuantKVCache, kv_quant_append, kv_quant_read

CODES = [torch.float8_e4m3fn, torch.int8]


def _rows(b, s, h, d, dtype, seed):
    """Rows of all sizes, with zeros, ties, borders of the exponent, subnormals."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, s, h, d, generator=g)
    x = x * torch.exp2(torch.randint(-20, 12, (b, s, h, 1), generator=g).float())
    x = x.to(dtype)
    flat = x.view(-1, d)
    n = len(flat)
    flat[0] = 0
    flat[1 % n, : d // 2] = 448.0
    flat[2 % n] = torch.arange(d).to(dtype) / 2 - d // 4        # halves: ties
    flat[3 % n] = 127.0
    flat[4 % n, 3] = torch.finfo(dtype).max
    flat[5 % n] = torch.finfo(dtype).smallest_normal / 4       # subnormal
    flat[6 % n, 0], flat[6 % n, 1:] = 448.5, 17.0
    flat[7 % n, 0] = 127.5
    return x


def _cache(b, h, room, d, code, dev, fill=7):
    codes = [torch.full((b, h, room, d), fill, dtype=torch.uint8, device=dev).view(code) for _ in "kv"]
    exps = [torch.full((b, h, room), 100, dtype=torch.uint8, device=dev) for _ in "kv"]
    return codes + exps


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("b,s,h,d", [(1, 1, 1, 64), (2, 9, 3, 128), (3, 5, 8, 64), (1, 70, 2, 256)])
def test_append_and_read(dev, dtype, code, b, s, h, d):
    room = s + 12
    k, v = _rows(b, s, h, d, dtype, 1), _rows(b, s, h, d, dtype, 2)
    c = _cache(b, h, room, d, code, dev)
    pos = torch.tensor([3, 0, 11][:b], dtype=torch.int32)
    kv_quant_append(k.to(dev), v.to(dev), *c, pos.to(dev))
    for x, codes, exps in ((k, c[0], c[2]), (v, c[1], c[3])):
        want, we = osp.quantise(x, code)
        codes, exps = codes.cpu(), exps.cpu()
        for i in range(b):
            p = int(pos[i])
            assert torch.equal(exps[i, :, p : p + s], we[i].T)
            assert torch.equal(codes[i, :, p : p + s].float(), want[i].transpose(0, 1).float())
            rest = torch.ones(room, dtype=torch.bool)
            rest[p : p + s] = False
            assert bool((codes[i].view(torch.uint8)[:, rest] == 7).all()), "rows beside were written"
            assert bool((exps[i][:, rest] == 100).all())
    for out in (torch.bfloat16, torch.float16):
        for got, codes, exps in zip(kv_quant_read(*c, room - 1, out), c[:2], c[2:]):
            want = osp.values(codes.cpu(), exps.cpu())[:, :, : room - 1]
            if out == torch.float16:
                want = want.clamp(-65504, 65504)
            assert got.dtype == out and torch.equal(got.cpu(), want.to(out))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_non_finite_rows(dev, code):
    """A row with an infinity or a NaN reads back as NaN, no other row does."""
    x = torch.randn(1, 4, 2, 64).bfloat16()
    x[0, 1, 0, 5], x[0, 2, 1, 63] = float("inf"), float("nan")
    c = _cache(1, 2, 16, 64, code, dev)
    kv_quant_append(x.to(dev), x.to(dev), *c, 0)
    k, _ = kv_quant_read(*c, 4)
    bad = torch.isnan(k.cpu())
    assert bool(bad[0, 0, 1].all()) and bool(bad[0, 1, 2].all()) and int(bad.sum()) == 2 * 64
    assert int((c[2].cpu() == 255).sum()) == 2


@pytest.mark.gpu
def test_append_edges(dev):
    """Positions before, across and past the cache, padded batches, strided
    inputs, an empty call, the cache of a larger batch, K and V apart."""
    b, s, h, d, room = 3, 4, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(b, s, 4 * h * d, generator=g).bfloat16()
    x = qkv.to(dev)
    k, v = x[..., : h * d].view(b, s, h, d), x[..., 2 * h * d : 3 * h * d].view(b, s, h, d)
    c = _cache(5, h, room, d, torch.int8, dev)
    part = [t[:b] for t in c]
    pos, cnt = torch.tensor([-2, 14, 6], dtype=torch.int32), torch.tensor([4, 4, 1], dtype=torch.int32)
    kv_quant_append(k, v, *part, pos.to(dev), cnt.to(dev))
    written = torch.zeros(5, room, dtype=torch.bool)
    written[0, 0:2] = written[1, 14:16] = True
    written[2, 6] = True
    for x, codes, exps in ((k, c[0], c[2]), (v, c[1], c[3])):
        want, we = osp.quantise(x.cpu(), torch.int8)
        codes, exps = codes.cpu(), exps.cpu()
        assert bool((codes.transpose(1, 2)[~written] == 7).all()) and bool((exps.transpose(1, 2)[~written] == 100).all())
        for i, p, n in ((0, -2, 4), (1, 14, 4), (2, 6, 1)):
            for j in range(n):
                if 0 <= p + j < room:
                    assert torch.equal(codes[i, :, p + j].double(), want[i, j]) and torch.equal(exps[i, :, p + j], we[i, j])
    before = [t.clone() for t in c]
    kv_quant_append(k[:, :0], v[:, :0], *part, 0)
    kv_quant_append(k, v, *part, 10 ** 9)
    assert all(torch.equal(a.view(torch.uint8), t.view(torch.uint8)) for a, t in zip(before, c))
    assert kv_quant_read(*part, 0)[0].shape == (b, h, 0, d)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_cache_object(dev, code):
    """QuantKVCache has KVCache's update contract on values that codes hold."""
    from torchplusplus_amd.llmops.kvcache import KVCache
    g = torch.Generator().manual_seed(4)
    plain = KVCache(21, 2, 64, torch.bfloat16, dev)
    cache = QuantKVCache(21, 2, 64, torch.bfloat16, dev, code_dtype=code)
    for s, index in ((5, None), (3, None), (4, 2), (1, 20)):
        # integers up to 7: held by either code exactly
        k, v = (torch.randint(-7, 8, (2, 2, s, 64), generator=g).bfloat16().to(dev) for _ in "kv")
        want, got = plain.update(k, v, index), cache.update(k, v, index)
        assert cache.cache_len == plain.cache_len
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="overflow"):
        cache.update(k, v, 21)
    with pytest.raises(ValueError):
        cache.append(k.transpose(1, 2), v.transpose(1, 2), -1)
    cache.reset()
    assert cache.cache_len == 0 and not bool(cache.read(21)[0].any())


@pytest.mark.gpu
def test_keep(dev):
    """The rows of an accepted path move behind the context, in both caches;
    nothing else moves, at the cache's end either."""
    from torchplusplus_amd.llmops.kvcache import KVCache
    b, h, room, d = 4, 2, 32, 64
    plain = KVCache(room, h, d, torch.bfloat16, dev, b)
    cache = QuantKVCache(room, h, d, torch.bfloat16, dev, b)
    x = torch.randint(-7, 8, (b, room, h, d)).bfloat16().to(dev)
    cache.append(x, x + 1, 0)
    plain.update(x.transpose(1, 2), (x + 1).transpose(1, 2))
    start = torch.tensor([3, 10, 0, 29], dtype=torch.int32, device=dev)
    path = torch.tensor([[0, 2, 5, -1], [1, 3, 4, 6], [-1, -1, -1, -1], [1, 2, -1, -1]], dtype=torch.int32, device=dev)
    want = x.clone()
    for i in range(b):
        for j in range(4):
            if path[i, j] >= 0:
                want[i, start[i] + j] = x[i, start[i] + path[i, j]]
    plain.keep(start, path)
    cache.keep(start, path)
    for k, v in ((plain.k_cache, plain.v_cache), cache.read(room)):
        assert torch.equal(k.transpose(1, 2), want) and torch.equal(v.transpose(1, 2), want + 1)


@pytest.mark.gpu
def test_captured(dev):
    """Append and read inside one graph, positions advanced between replays."""
    b, s, h, d, room = 2, 3, 2, 128, 32
    x = torch.randn(b, s, h, d, device=dev).bfloat16()
    c, e = _cache(b, h, room, d, torch.int8, dev), _cache(b, h, room, d, torch.int8, dev)
    pos = torch.zeros(b, dtype=torch.int32, device=dev)
    kv_quant_append(x, x, *e, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_quant_append(x, x, *c, pos)
        got = kv_quant_read(*c, room)
    for i in range(3):
        pos.fill_(4 * i)
        x.normal_()
        graph.replay()
        kv_quant_append(x, x, *e, 4 * i)
        want = kv_quant_read(*e, room)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals_on_the_host():
    with pytest.raises(TypeError):
        QuantKVCache(16, 2, 64, code_dtype=torch.uint8)
    with pytest.raises(TypeError):
        QuantKVCache(16, 2, 64, dtype=torch.float32)
    with pytest.raises(ValueError):
        QuantKVCache(16, 2, 80)
    c = QuantKVCache(16, 2, 64, device="cpu", batch_size=1)
    assert c.k_codes.shape == (1, 2, 16, 64) and c.k_codes.dtype == torch.float8_e4m3fn
    assert QuantKVCache(17, 2, 64, device="cpu", batch_size=1).k_exps.shape == (1, 2, 32)
    with pytest.raises(ValueError, match="overflow"):
        c.ensure(1, 17)
    k = torch.zeros(1, 1, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.append(k, k, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.read(3)
    with pytest.raises(TypeError):
        kv_quant_read(c.k_codes, c.v_codes, c.k_exps, c.v_exps, 3, torch.float32)
    with pytest.raises(TypeError):
        kv_quant_append(k, k, k, k, c.k_exps, c.v_exps, 0)


@pytest.mark.gpu
def test_refusals(dev):
    c = _cache(2, 2, 16, 64, torch.int8, dev)
    k = torch.zeros(2, 3, 2, 64, dtype=torch.float16, device=dev)
    pos = torch.zeros(2, dtype=torch.int32, device=dev)
    odd = torch.zeros(2 * 3 * 2 * 64 + 1, dtype=torch.float16, device=dev)[1:].view(2, 3, 2, 64)
    for bad in ((k, k.bfloat16(), *c, pos), (k, k[:, :2], *c, pos), (k[:1], k[:1], *c, pos),
                (k, k, *c, pos.long()), (k, k, *c, pos[:1]), (k, k, c[0], c[1][:, :, :8], *c[2:], pos),
                (k, k, c[0], c[1].view(torch.float8_e4m3fn), *c[2:], pos), (k, k, *c[:2], c[2][:, :, 1:], c[3], pos),
                (odd, odd, *c, pos), (k, k, c[0], c[0], *c[2:], pos), (k, k, *c[:2], c[2], c[2], pos), (k.float(), k.float(), *c, pos), (k, k, *c, pos.cpu())):
        with pytest.raises(RuntimeError):
            kv_quant_append(*bad)
    with pytest.raises(RuntimeError):
        kv_quant_read(*c, 17)
    with pytest.raises(RuntimeError):
        kv_quant_read(*c, -1)


@pytest.mark.gpu
def test_append_refuses_rows_that_sequences_share(dev):
    c = _cache(1, 2, 16, 64, torch.int8, dev)
    k = torch.zeros(2, 3, 2, 64, dtype=torch.float16, device=dev)
    shared = [x.expand(2, *x.shape[1:]) for x in c]
    with pytest.raises(RuntimeError, match="of their own"):
        kv_quant_append(k, k, *shared, 0)
    assert kv_quant_read(*shared, 5)[0].shape == (2, 2, 5, 64)  # reading a shared prompt is fine
