"""packed_attention of a few queries a sequence behind cached keys, where the query heads of a
group share a tile."""
import math

import pytest
import torch

from tests.test_packed_attention import check, ends, i32, make


def both(n):
    return [1 + (5 * i) % n for i in range(7)], [40 + (137 * i) % 500 for i in range(7)]


CASES = [([1] * 5, [700, 1, 64, 333, 2000]), ([4, 4, 4], [3000, 4, 9]), ([3, 0, 1, 9, 2], [50, 20, 0, 4, 130]), both(9), both(16), both(30),
         ([1] * 300, [1 + (7 * i) % 90 for i in range(300)]), ([2, 1, 5] * 40, [30, 100, 65] * 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(8, 4, 128), (8, 2, 64), (8, 1, 128), (16, 1, 64), (64, 2, 128), (6, 2, 128), (12, 1, 64), (10, 5, 64)])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_lengths(dev, i, hq, hk, d, dtype):
    from torchplusplus_amd.attention import packed_attention
    lq, lk = CASES[i]
    q, k, v = make(lq, lk, hq, hk, d, dtype, i, dev)
    cu, cuk = ends(lq), ends(lk)
    check(packed_attention(q, k, v, i32(cu, dev), i32(cuk, dev)), q, k, v, cu, cuk)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk,d", [(16, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("causal,window", [(True, (20, -1)), (False, (-1, -1)), (False, (5, 3)), (False, (100, -1))])
def test_windows_strides_and_rows_of_no_sequence(dev, hq, hk, d, causal, window):
    from torchplusplus_amd.attention import packed_attention
    lq, lk = [1, 7, 2, 12, 0, 3], [300, 150, 1, 70, 9, 64]
    q, k, v = make(lq, lk, hq, hk, d, torch.float16, 3, dev)
    cu, cuk = ends(lq), ends(lk)
    n = len(q) + 8  # rows ahead of the first sequence and behind the last; heads outermost
    wide = torch.full((hq, n, d + 8), 9.0, dtype=q.dtype, device=dev).transpose(0, 1)[..., :d]
    wide[3:-5] = q
    out = torch.full((hq, n, d + 16), 7.0, dtype=q.dtype, device=dev).transpose(0, 1)[..., :d]
    at = i32([x + 3 for x in cu], dev)
    kw = dict(causal=causal, window_size=window)
    got = packed_attention(wide, k, v, at, i32(cuk, dev), out=out, **kw)
    check(got[3:-5], q, k, v, cu, cuk, causal=causal, window=window)
    assert (got[:3] == 7).all() and (got[-5:] == 7).all()
    new = packed_attention(wide, k, v, at, i32(cuk, dev), **kw)
    assert torch.equal(new[3:-5], got[3:-5]) and (new[:3] == 0).all() and (new[-5:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [2, 60])
def test_values_that_are_not_finite_where_they_are_not_seen(dev, batch):
    """In keys behind a query of its own sequence: its other rows' results stay, head by head."""
    from torchplusplus_amd.attention import packed_attention
    lq, lk = [4] * batch, [70] * batch
    q, k, v = make(lq, lk, 8, 2, 64, torch.bfloat16, 5, dev)
    cu, cuk = i32(ends(lq), dev), i32(ends(lk), dev)
    want = packed_attention(q, k, v, cu, cuk)
    for row, x in ((68, math.inf), (69, math.nan)):  # seen by the last two queries, and by the last
        k[row], v[row, 0] = x, x
    got = packed_attention(q, k, v, cu, cuk)
    assert (got[:2].float() - want[:2].float()).abs().max() <= 2 * 2.0 ** -8 * want[:2].float().abs().max()
    assert torch.equal(got[4:], want[4:]) and got[3].isnan().all() and not got[2].isfinite().all()
