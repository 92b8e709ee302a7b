"""tree_attention's weights: how many bits of them count, and how small they may be.

Scores here are exact: queries are one-hot, so a score is one element of a key. A
weight's relative error is then that of its exponent x = s log2(e), two roundings of
2^-24 |x| (the scale, the product) times ln 2, and 2^-23 of the exponential: at most
(2 ln 2 |x| + 2) 2^-24."""
import math

import numpy as np
import pytest
import torch

from oracle import speculative as osp
from tests.test_tree_attention import CODES

# B, T, Hq, Hkv, D: one token, 16 rows, 32 rows, more rows (of a KV head); head sizes
# 64 and 128 on the matrix cores, 96 not
SHAPES = [(1, 1, 2, 2, 128), (2, 4, 4, 2, 64), (1, 8, 4, 2, 128), (1, 16, 4, 2, 64), (1, 16, 4, 2, 128),
          (1, 12, 8, 1, 64), (1, 33, 8, 1, 128), (1, 2, 2, 1, 96)]


def make(shape, scores, values, dtype, code, dev):
    """q, cache, its exponents and its values: key j of every head has score scores[j]
    and value values[j] throughout (softmax scale 1)."""
    b, t, hq, hkv, d = shape
    room = len(scores)
    q = torch.zeros(b, t, hq, d, dtype=dtype)
    q[..., 0] = 1
    k, v = torch.zeros(b, hkv, room, d), torch.zeros(b, hkv, room, d)
    k[..., 0], v[:] = torch.tensor(scores), torch.tensor(values).unsqueeze(-1)
    if code is None:
        assert torch.equal(k.to(dtype).float(), k) and torch.equal(v.to(dtype).float(), v)
        return q.to(dev), [x.to(dtype).to(dev) for x in (k, v)], {}
    both = [osp.quantise(x, code) for x in (k, v)]
    for (c, e), x in zip(both, (k, v)):
        assert torch.equal(osp.values(c, e), x.double()), "the codes do not hold the inputs"
    return (q.to(dev), [c.float().to(code).to(dev) for c, _ in both],
            dict(k_exps=both[0][1].to(dev), v_exps=both[1][1].to(dev)))


@pytest.mark.gpu
@pytest.mark.parametrize("drop", [20.0, 26.0, 28.0, 30.0])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_weights_of_large_values(dev, dtype, code, shape, drop):
    """One key in 32 has weight 1 and value 0, the others exp(-drop) (down to 2^-43)
    and value 57344: the result is made of the small weights alone. Tolerance: the
    output's rounding and the weights' error (|x| at most 30 log2(e) = 43.3: 62 units
    of 2^-24 at the exponent; 2^-20 covers what a sum of 704 such terms loses, n / 32
    roundings of 2^-24 a wave and 96 inside of each product, and P's own 2^-21)."""
    from torchplusplus_amd.attention import tree_attention
    n = 704
    room = n + 64
    scores = [0.0 if j % 32 == 0 else -drop for j in range(room)]
    values = [0.0 if j % 32 == 0 else 57344.0 for j in range(room)]
    b, t = shape[:2]
    q, cache, kw = make(shape, scores, values, dtype, code, dev)
    par = torch.full((b, t), -1, dtype=torch.int32)
    lens = torch.full((b,), n, dtype=torch.int32)
    got = tree_attention(q, *cache, lens.to(dev), par.to(dev), softmax_scale=1.0, **kw).double().cpu()
    for i in range(t):
        keys = list(range(n)) + [n + i]
        w = [math.exp(scores[j]) for j in keys]
        want = sum(x * values[j] for x, j in zip(w, keys)) / sum(w)
        tol = torch.finfo(dtype).eps / 2 * want * 1.01 + 2.0 ** -25 + (62 * 2.0 ** -24 + 2.0 ** -20) * want
        off = (got[:, i] - want).abs().max()
        assert float(off) <= tol, f"token {i}: {float(got[:, i].min())} .. {float(got[:, i].max())}, not {want}"


def cut(x):
    """The upper half of a float's bits: a bfloat16, not rounded."""
    return float((np.float32(x).view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32))


def low_bits():
    """A score -m / 32 that each code holds (m below 16), whose weight is furthest from
    the sum of two such halves: 2^-16 of itself or more."""
    best = (0.0, 0)
    for m in range(8, 16):
        w = float(np.float32(math.exp(-m / 32)))
        best = max(best, ((w - cut(w) - cut(w - cut(w))) / w, m))
    assert best[0] > 2.0 ** -16
    return -best[1] / 32


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_weights_keep_their_bits(dev, dtype, code, shape):
    """Keys of weight 1 and value 1 against keys of weight w and value -1, so many of
    each that they all but cancel: what is left shows the weights' error, which weights
    of 16 bits would not pass and weights of 8 by far. Runs of each kind are short, so
    that partial sums stay below 16. Tolerance: the output's rounding, half of the
    mass times a weight's error (|x| < 0.5: 3 units of 2^-24), and the sums: at most
    96 roundings (32 keys in three parts) of 2^-24 of a partial sum a batch of 32
    keys, whose mass is at least 24: 96 * 16 / 24 units."""
    from torchplusplus_amd.attention import tree_attention
    s = low_bits()
    w = math.exp(s)
    scores, values, total = [], [], 0.0
    while len(scores) < 1600:
        if total <= 0:
            scores, values, total = scores + [0.0], values + [1.0], total + 1.0
        else:
            scores, values, total = scores + [s], values + [-1.0], total - w
    # the length, past 1400, at which the sum is least; the drafted keys behind it are
    # worth nothing
    sums = np.cumsum([math.exp(a) * v for a, v in zip(scores, values)])
    b, t = shape[:2]
    n = 1401 + int(np.argmin(np.abs(sums[1400:1535])))
    scores[n:], values[n:] = [-16.0] * (1600 - n), [0.0] * (1600 - n)
    want = sums[n - 1] / (sum(math.exp(x) for x in scores[:n]) + math.exp(-16))
    q, cache, kw = make(shape, scores, values, dtype, code, dev)
    par = torch.full((b, t), -1, dtype=torch.int32)  # each sees the context and itself
    lens = torch.full((b,), n, dtype=torch.int32)
    got = tree_attention(q, *cache, lens.to(dev), par.to(dev), softmax_scale=1.0, **kw).double().cpu()
    tol = torch.finfo(dtype).eps / 2 * abs(want) * 1.01 + 2.0 ** -25 + (1.5 + 96 * 16 / 24) * 2.0 ** -24
    off = float((got - want).abs().max())
    assert off <= tol, f"off by {off}, {tol} allowed, of {want}"
