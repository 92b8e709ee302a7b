"""token_logprobs against the 64-bit form in oracle/serving.py.

Tolerances. The sum Z of V terms e^d, d = x - max: a thread adds V / 256 of them one
after the other, in chunks that are merged by trees, each step 2^-24 of the sum; a term's
own error is 2 |d| + 4 units of 2^-24 (the exponent's product, the exponential), on
the average over the terms' shares 2 H + 4; changes of the maximum rescale at most V /
2048 + 20 times, 4 units each. So Z, and with it ln Z, is off by u = (V / 256 + V / 512 +
100 + 2 H) 2^-24 at most; the logarithm, the difference x - max and their sum add units of
|result| and |x - max|. The entropy's second term is a mean of the same terms: H (2 u)."""
import math

import pytest
import torch

from oracle import serving as oracle

U = 2.0 ** -24


def check(r, logits, tokens, top):
    lp, ent, best, ids = oracle.logprobs(logits, tokens, top)
    v = logits.shape[1]
    x = logits.double().cpu()
    far = (x.amax(1) - x.gather(1, tokens.cpu().clamp(0, v - 1).unsqueeze(1)).squeeze(1)).nan_to_num(0, 0, 0)
    u = (v / 256 + v / 512 + 100 + 2 * ent.nan_to_num(0)) * U

    def near(got, want, tol, what):
        got = got.double().cpu()
        same = (got == want) | (got.isnan() & want.isnan())
        bad = ~(same | ((got - want).abs() <= tol))
        assert not bad.any(), (what, bad.nonzero()[:3].tolist(), got[bad][:3], want[bad][:3])

    near(r.logprobs, lp, u + 4 * U * (lp.abs() + far), "logprobs")
    near(r.entropy, ent, u + (2 * u + 8 * U) * ent.nan_to_num(0), "entropy")
    if top:
        assert torch.equal(r.top_tokens.cpu(), ids)
        near(r.top_logprobs, best, u.unsqueeze(1) + 8 * U * best.abs(), "top")
    else:
        assert r.top_logprobs is None and r.top_tokens is None


def rows(n, v, dtype, seed, dev, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, v, generator=g) * spread).to(dtype).to(dev)
    return x, torch.randint(0, v, (n,), generator=g).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,v", [(1, 1), (3, 2), (2, 7), (5, 100), (4, 255), (3, 2047), (2, 2048), (3, 2049), (7, 4097), (2, 50257),
                                 (1, 151936), (9, 32000)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_sizes(dev, n, v, dtype, top):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    x, t = rows(n, v, dtype, v + n, dev)
    check(token_logprobs(x, t, min(top, v)), x, t, min(top, v))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 600, 1500])
def test_many_rows(dev, n, dtype):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    x, t = rows(n, 3001, dtype, n, dev, spread=5.0)
    check(token_logprobs(x, t, 7), x, t, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 700])
def test_orders_ties_and_places(dev, n):
    """Rising, falling and constant rows, few distinct values, the largest in one thread's
    or one run's places, zeros of both signs: ties go to the lowest index."""
    from torchplusplus_amd.llmops.scoring import token_logprobs
    v = 20000
    i = torch.arange(v, dtype=torch.float32)
    kinds = [i / 1000, -i / 1000, torch.zeros(v), (i % 7), (i % 2048 < 8).float() * (20 - i / v), (i % 2048 < 256) * (30 + i / v),
             torch.where(i % 3 == 0, 0.0, -0.0), -torch.floor(i / 9), (i == v - 1).float(), i * 0 - 3e38, (i >= v - 40) * 5.0]
    x = torch.stack([kinds[r % len(kinds)] for r in range(max(n, len(kinds)))]).to(dev)
    t = torch.arange(len(x), device=dev) * 1237 % v
    for top in (1, 20, 32):
        check(token_logprobs(x, t, top), x, t, top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("copies", [1, 200])
def test_masked_and_not_finite(dev, dtype, copies):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    v = 5000
    x, t = rows(8, v, dtype, 3, dev)
    low = torch.finfo(dtype).min
    x[0, 3:] = -math.inf                # three left, fewer than asked for
    x[1] = -math.inf
    x[1, 4321] = 2.0                    # one left
    x[2] = -math.inf                    # none
    x[3, 17] = math.nan
    x[4, 4999] = math.inf
    x[5, :4000] = low
    x[6] = low
    x[7, 100], x[7, 200] = math.nan, math.inf
    x, t = x.repeat(copies, 1), t.repeat(copies)
    t[0], t[1] = 1, 4321
    check(token_logprobs(x, t, 9), x, t, 9)


@pytest.mark.gpu
def test_padding_strides_and_shapes(dev):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    x, t = rows(6, 1000, torch.bfloat16, 4, dev)
    t[1], t[2], t[3] = -1, 1000, -100
    r = token_logprobs(x, t, 3)
    check(r, x, t, 3)
    assert (r.logprobs[1:4] == 0).all()
    wide = torch.zeros(6, 1203, dtype=x.dtype, device=dev)
    wide[:, 101:1101] = x
    for y in (wide[:, 101:1101], wide[:, 101:1101].view(6, 1000)):
        s = token_logprobs(y, t, 3)
        assert all(torch.equal(a, b) for a, b in zip(s, r))
    s = token_logprobs(x.view(2, 3, 1000), t.view(2, 3), 3)
    assert s.logprobs.shape == (2, 3) and s.top_tokens.shape == (2, 3, 3)
    assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(s, r))
    one = token_logprobs(x[0], t[0], 2)
    assert one.logprobs.shape == () and one.top_logprobs.shape == (2,) and torch.equal(one.logprobs, r.logprobs[0])
    same = token_logprobs(x[:1].expand(4, 1000), t[:4])
    check(same, x[:1].expand(4, 1000), t[:4], 0)
    none = token_logprobs(x[:0], t[:0], 2)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 8, 900])
def test_streams_and_graphs(dev, n):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    x, t = rows(n, 32000, torch.bfloat16, 5, dev)
    want = token_logprobs(x, t, 5)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(token_logprobs(x, t, 5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, t, 5)
        out2 = token_logprobs(x, t, 5)
    for step in range(4):
        x.copy_(x.roll(777, 1))
        want = token_logprobs(x, t, 5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(out, want, out2))


@pytest.mark.gpu
def test_refusals(dev):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    x, t = rows(3, 50, torch.float16, 0, dev)
    for args in ((x.double(), t), (x, t.int()), (x, t.cpu()), (x.cpu(), t.cpu()), (x, t, 33), (x, t, 51), (x, t, -1),
                 (x.t().contiguous().t(), t), (x[:, :0], t)):
        with pytest.raises(RuntimeError):
            token_logprobs(*args)
    with pytest.raises(ValueError):
        token_logprobs(x, t[:2])
