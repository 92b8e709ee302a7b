"""tree_attention where scores or values are infinite or near the type's end: every
kernel (the sizes of test_tree_precision.py) answers as the formula does. Queries are
one-hot and the scale is 1, so that a score is one element of a key, exactly."""
import math

import pytest
import torch

from tests.test_tree_attention import CODES
from tests.test_tree_precision import SHAPES, make

INF = math.inf


def attend(dev, shape, scores, values, dtype, code, n, par):
    from torchplusplus_amd.attention import tree_attention
    q, cache, kw = make(shape, scores, values, dtype, code, dev)
    lens = torch.full((shape[0],), n, dtype=torch.int32)
    return tree_attention(q, *cache, lens.to(dev), par.to(dev), softmax_scale=1.0, **kw).float().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", [20, 704])
def test_scores_of_minus_infinity(dev, dtype, shape, n):
    """All visible scores -inf: NaN, as the softmax of such a row is. One finite score
    among them: its value. A token that sees nothing: 0."""
    b, t = shape[:2]
    scores, values = [-INF] * (n + 64), [3.0] * (n + 64)
    par = torch.full((b, t), -1, dtype=torch.int32)
    finite = t - 1 if t > 1 else None  # the last token's own key
    if finite is not None:
        scores[n + finite], values[n + finite] = 1.0, 7.0
    if t > 2:
        par[:, 1] = -2
    o = attend(dev, shape, scores, values, dtype, None, n, par)
    for i in range(t):
        if t > 2 and i == 1:
            assert bool((o[:, i] == 0).all())
        elif i == finite:
            assert bool((o[:, i] == 7.0).all())
        else:
            assert bool(torch.isnan(o[:, i]).all()), f"token {i}: {o[0, i, 0, :4]}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n,at", [(20, 5), (704, 3), (704, 600)])
def test_infinite_values_in_the_context(dev, dtype, shape, n, at):
    """A value of infinity that all tokens see, of any weight above 0: infinity of its
    sign; two of opposite signs: NaN."""
    b, t = shape[:2]
    g = torch.Generator().manual_seed(at)
    par = torch.full((b, t), -1, dtype=torch.int32)
    scores = (torch.randint(-32, 33, (n + 64,), generator=g).float() / 16).tolist()
    scores[1] = 3.0
    for where in (at, 1):  # some weight, and the largest
        values = torch.randint(-3, 4, (n + 64,), generator=g).float().tolist()
        values[where] = -INF
        assert bool((attend(dev, shape, scores, values, dtype, None, n, par) == -INF).all())
        values[where + 7] = INF
        assert bool(torch.isnan(attend(dev, shape, scores, values, dtype, None, n, par)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_nan_scores_and_values(dev, dtype, shape):
    """A NaN among the scores of the context: NaN for all; in a drafted token's key or
    value: for those that see it alone."""
    from torchplusplus_amd.attention import tree_attention
    b, t = shape[:2]
    n = 300
    par = torch.full((b, t), -1, dtype=torch.int32)
    for where in (70, n):
        for which in (0, 1):
            q, cache, _ = make(shape, [0.5] * (n + 64), [2.0] * (n + 64), dtype, None, dev)
            cache[which][:, :, where, 0 if which == 0 else slice(None)] = math.nan
            lens = torch.full((b,), n, dtype=torch.int32, device=dev)
            o = tree_attention(q, *cache, lens, par.to(dev), softmax_scale=1.0).float().cpu()
            assert bool(torch.isnan(o[:, 0]).all())
            assert bool(torch.isnan(o[:, 1:]).all()) if where < n else bool((o[:, 1:] == 2.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("t,hq,d", [(1, 1, 128), (4, 2, 64), (16, 2, 128), (33, 1, 64), (12, 4, 128), (1, 1, 96)])
def test_values_near_the_end_of_bfloat16(dev, code, t, hq, d):
    """One value of 2^126 among keys whose scores rise by less than 8 log(2) along a
    wave's tiles (512 pairs: one block has all of a pair's keys): weights above 1 would
    leave fp32's range. Tolerance: the output's rounding, the weights' error, (2 ln 2 *
    7.3 + 2) 2^-24, and the roundings of their sum, 10 tiles and 32 a tile: 2^-18."""
    from torchplusplus_amd.attention import tree_attention
    b, hkv, n = 64, 8, 300
    scores = [0.0] * 160 + [5.0] * (n - 96)
    values = [0.0] * (n + 64)
    values[n - 10] = 2.0 ** 126
    q, cache, kw = make((1, t, hq, 1, d), scores, values, torch.bfloat16, code, dev)
    spread = lambda x: x.view(torch.uint8).expand(b, hkv, *x.view(torch.uint8).shape[2:]).contiguous().view(x.dtype)  # noqa: E731
    q = q.repeat(b, 1, hkv, 1)
    cache, kw = [spread(x) for x in cache], {k: spread(x) for k, x in kw.items()}
    par, lens = torch.full((b, t), -1, dtype=torch.int32), torch.full((b,), n, dtype=torch.int32)
    o = tree_attention(q, *cache, lens.to(dev), par.to(dev), softmax_scale=1.0, **kw).double().cpu()
    want = 2.0 ** 126 * math.exp(5.0) / (160 + (n - 159) * math.exp(5.0))
    assert bool(((o - want).abs() <= (2.0 ** -9 + 2.0 ** -18) * want).all()), (float(o.min()), float(o.max()), want)
