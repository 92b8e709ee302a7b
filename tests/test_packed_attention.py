"""packed_attention against the 64-bit form in oracle/serving.py.

Tolerance of an element o = sum w v, with A = sum w |v| (the oracle's second result):
its own rounding eps / 2 |o| (half the least fp16 step, 2^-25), the rounding of the
weights to the matrix cores' type, eps / 2 of each, fp16 weights below 2^-24 of a scale
of 2^7 cut (2^-32 of |v| a key), and fp32 arithmetic: a score's error is at most (D + 8)
2^-24 of sum |q k| scale (the third result, which bounds |score| too) plus 2^-22, twice
that as relative error of a weight and again of their sum, and sums over n keys n 2^-24
A."""
import math

import pytest
import torch

from oracle import serving as oracle


def tolerance(o, mean, size, dtype, n, d, vmax):
    half = torch.finfo(dtype).eps / 2
    fp32 = 4 * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -22) + 2 * n * 2.0 ** -24
    cut = n * 2.0 ** -32 * vmax if dtype == torch.float16 else 0.0
    return half * o.abs() * (1 + 2 * half) + 2.0 ** -25 + (half + fp32) * mean + cut


def make(lens, lens_k, hq, hk, d, dtype, seed, dev, extra=0):
    g = torch.Generator().manual_seed(seed)
    n, nk = sum(lens) + extra, sum(lens_k) + (extra if lens_k is lens else 0)
    q, k, v = (torch.randn(m, h, d, generator=g).to(dtype).to(dev) for m, h in ((n, hq), (nk, hk), (nk, hk)))
    return q, k, v


def ends(lens, first=0):
    out = [first]
    for x in lens:
        out.append(out[-1] + x)
    return out


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def check(got, q, k, v, cu, cu_k, **kw):
    o, mean, size = oracle.packed_attention(q, k, v, cu, cu_k, **kw)
    d, n = q.shape[2], min(max([b - a for a, b in zip(cu_k, cu_k[1:])], default=0), len(k))
    tol = tolerance(o, mean, size, q.dtype, n, d, float(v.abs().max().float()) if v.numel() else 0.0)
    err = (got.double().cpu() - o).abs()
    assert torch.isfinite(got).all()
    bad = err > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((err / tol).max()))


LENS = [[1], [2, 0, 3], [31, 32, 33, 1], [64, 63, 65], [127, 128, 129], [5, 300, 1, 77], [0, 0, 200, 0], [513],
        [1] * 70, [257, 30, 256, 255, 3]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (4, 4, 64), (8, 1, 128), (6, 2, 64), (3, 1, 80)])
@pytest.mark.parametrize("i", range(len(LENS)))
def test_lengths(dev, i, hq, hk, d, dtype):
    from torchplusplus_amd.attention import packed_attention
    q, k, v = make(LENS[i], LENS[i], hq, hk, d, dtype, i, dev)
    cu = ends(LENS[i])
    check(packed_attention(q, k, v, i32(cu, dev)), q, k, v, cu, cu)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (2, 2, 64), (2, 1, 256)])
@pytest.mark.parametrize("causal,window", [(True, (-1, -1)), (True, (0, -1)), (True, (40, 7)), (False, (-1, -1)),
                                           (False, (5, 3)), (False, (-1, 0)), (False, (100, -1)), (True, (2 ** 31 - 1, -1)),
                                           (False, (2 ** 40, 2 ** 40))])
def test_windows_and_key_lengths(dev, hq, hk, d, causal, window):
    """More keys than queries, fewer (rows that see nothing), none at all."""
    from torchplusplus_amd.attention import packed_attention
    lq, lk = [3, 150, 40, 1, 17, 0, 70], [400, 150, 9, 200, 0, 30, 64]
    q, k, v = make(lq, lk, hq, hk, d, torch.bfloat16, 7, dev)
    cu, cuk = ends(lq), ends(lk)
    got = packed_attention(q, k, v, i32(cu, dev), i32(cuk, dev), causal=causal, window_size=window)
    check(got, q, k, v, cu, cuk, causal=causal, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_and_short_together(dev, dtype):
    from torchplusplus_amd.attention import packed_attention
    lens = [1500, 9, 700, 1, 64]
    q, k, v = make(lens, lens, 4, 2, 128, dtype, 3, dev)
    cu = ends(lens)
    check(packed_attention(q, k, v, i32(cu, dev)), q, k, v, cu, cu)
    # many tiles: as many as fill the card more than once, heads of one KV head each
    lens = [600, 1, 257, 900, 33] * 3
    q, k, v = make(lens, lens, 16, 8, 64, dtype, 4, dev)
    cu = ends(lens)
    check(packed_attention(q, k, v, i32(cu, dev)), q, k, v, cu, cu)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 72])
def test_strides_scale_and_out(dev, d):
    from torchplusplus_amd.attention import packed_attention
    lens = [70, 5, 130]
    n, hq, hk = sum(lens), 4, 2
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(torch.float16).to(dev)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], 1))
    cu = ends(lens)
    check(packed_attention(q, k, v, i32(cu, dev), softmax_scale=0.3), q, k, v, cu, cu, scale=0.3)
    # heads ahead of tokens; an out of its own layout
    qt, kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    out = torch.full((hq, n, d), 7.0, dtype=q.dtype, device=dev).transpose(0, 1)
    assert packed_attention(qt, kt, vt, i32(cu, dev), out=out).data_ptr() == out.data_ptr()
    check(out, q, k, v, cu, cu)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 40])
def test_rows_of_no_sequence(dev, d):
    """Ahead of the first and behind the last: left as they were, 0 in a new tensor; ends
    past the tensors are cut."""
    from torchplusplus_amd.attention import packed_attention
    lens = [40, 3, 90]
    q, k, v = make(lens, lens, 4, 2, d, torch.bfloat16, 5, dev, extra=75)
    cu = ends(lens, 2)
    got = packed_attention(q, k, v, i32(cu, dev))
    check(got, q, k, v, cu, cu)
    assert (got[:2] == 0).all() and (got[cu[-1]:] == 0).all()
    out = torch.full_like(q, 5.0)
    packed_attention(q, k, v, i32(cu, dev), out=out)
    assert torch.equal(out[2 : cu[-1]], got[2 : cu[-1]])
    assert (out[:2] == 5).all() and (out[cu[-1]:] == 5).all()
    far = cu[:-1] + [1 << 30]
    check(packed_attention(q, k, v, i32(far, dev)), q, k, v, far, far)
    low = [-2 ** 31] + cu[1:]
    check(packed_attention(q, k, v, i32(low, dev)), q, k, v, low, low)
    empty = packed_attention(q, k, v, i32([0], dev))
    assert (empty == 0).all()
    assert packed_attention(q[:0], k, v, i32([0, 0], dev), i32([0, 9], dev)).shape == (0, 4, d)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_not_finite_where_they_are_not_seen(dev, d, dtype):
    """Infinities and NaN among the keys and values of later tokens, of the neighbouring
    sequences and behind the last leave every row that does not see them alone."""
    from torchplusplus_amd.attention import packed_attention
    lens = [37, 100, 64, 9]
    q, k, v = make(lens, lens, 4, 2, d, dtype, 9, dev, extra=10)
    cu = ends(lens)
    want = packed_attention(q, k, v, i32(cu, dev))
    k2, v2 = k.clone(), v.clone()
    bad = [36, 36 + 100, 90, 200, cu[-1], cu[-1] + 3]  # last ones of 0 and 1, inside 1 and 2, behind
    for r, x in zip(bad, (math.nan, math.inf, -math.inf, math.nan, math.inf, math.nan)):
        k2[r], v2[r] = x, x
    got = packed_attention(q, k2, v2, i32(cu, dev))
    o, mean, size = oracle.packed_attention(q, k2, v2, cu, cu)
    clean = torch.isfinite(o).all(-1).to(dev)
    assert clean[:36].all() and clean[37:90].all() and not clean[90:137].any() and not clean[36].any()
    tol = tolerance(o, mean, size, dtype, 100, d, 8.0).to(dev)
    err = (got.double() - o.to(dev)).abs()
    assert (err <= tol)[clean].all()
    assert not torch.isfinite(got)[~clean].all(-1).any()
    assert torch.isfinite(want[:cu[-1]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 40])
def test_scores_of_minus_infinity(dev, d):
    from torchplusplus_amd.attention import packed_attention
    lens = [70, 40]
    q, k, v = make(lens, lens, 2, 1, d, torch.bfloat16, 2, dev)
    q = q.abs() + 0.1
    k[:70] = -math.inf  # every score of the first sequence
    got = packed_attention(q, k, v, i32(ends(lens), dev))
    assert torch.isnan(got[:70]).all() and torch.isfinite(got[70:]).all()
    k[3] = 1.0          # rows 3 .. 69 have one key left
    got = packed_attention(q, k, v, i32(ends(lens), dev))
    assert torch.isnan(got[:3]).all() and torch.equal(got[3:70], v[3:4].expand(67, 2, d))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scores_that_rise_and_fall_and_large_values(dev, d, dtype):
    """A maximum that moves with every key, or stands in the first; values near the
    types' ends stay finite."""
    from torchplusplus_amd.attention import packed_attention
    n = 500
    g = torch.Generator().manual_seed(8)
    q = torch.ones(n, 2, d).to(dtype).to(dev)
    big = 2.0 ** 15 if dtype == torch.float16 else 2.0 ** 126
    v = ((torch.rand(n, 2, d, generator=g) + 0.5) * big).to(dtype).to(dev)
    for slope in (0.5, -0.5, 0.0):
        k = (torch.arange(n).view(n, 1, 1) * slope / d ** 0.5 * torch.ones(n, 2, d)).to(dtype).to(dev)
        cu = [0, n]
        check(packed_attention(q, k, v, i32(cu, dev)), q, k, v, cu, cu)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[200, 3, 80], [700, 1000, 1, 300]])
def test_streams_and_graphs(dev, lens):
    """On a side stream and captured: replayed with other lengths in the same buffers,
    eager work between the replays, each against the eager call."""
    from torchplusplus_amd.attention import packed_attention
    q, k, v = make(lens, lens, 16, 8, 128, torch.bfloat16, 6, dev)
    cu = i32(ends(lens), dev)
    want = packed_attention(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = packed_attention(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(q, k, v, cu)
        out2 = packed_attention(q, k, v, cu)
    total = sum(lens)
    for cut in (list(lens), [total - 7, 0, 7], [1, total - 1], [total]):
        cu.copy_(i32((ends(cut) + [total] * len(lens))[: len(lens) + 1], dev))
        want = packed_attention(q, k, v, cu)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want)


@pytest.mark.gpu
def test_refusals(dev):
    from torchplusplus_amd.attention import packed_attention
    q, k, v = make([9, 4], [9, 4], 4, 2, 64, torch.float16, 0, dev)
    cu = i32([0, 9, 13], dev)
    for args, kw in (((q.float(), k.float(), v.float(), cu), {}), ((q, k.bfloat16(), v, cu), {}), ((q[None], k, v, cu), {}),
                     ((q, k[:, :, :32], v[:, :, :32], cu), {}), ((q[:, :3], k, v, cu), {}), ((q, k, v[:5], cu), {}),
                     ((q, k[:5], v[:5], cu), {}), ((q, k, v, cu.long()), {}), ((q, k, v, cu.cpu()), {}),
                     ((q, k, v, cu[:0]), {}), ((q, k, v, cu, cu[:2]), {}), ((q.cpu(), k, v, cu), {}),
                     ((q, k, v, cu), {"out": q}), ((q, k, v, cu), {"out": torch.empty_like(q)[:5]}),
                     ((q, k, v, cu), {"out": torch.empty(1, 4, 64, dtype=q.dtype, device=dev).expand(13, 4, 64)})):
        with pytest.raises(RuntimeError):
            packed_attention(*args, **kw)


@pytest.mark.parametrize("scale", [0.0, -1.0, math.nan, math.inf])
def test_refuses_a_scale_that_is_not_above_0(scale):
    from torchplusplus_amd.attention import packed_attention
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="softmax_scale"):
        packed_attention(x, x, x, torch.zeros(2, dtype=torch.int32), softmax_scale=scale)
