"""paged_attention against the 64-bit form in oracle/serving.py. Tolerance: that of
test_packed_attention.py, whose terms are the same."""
import math

import pytest
import torch

from oracle import serving as oracle
from tests.test_packed_attention import i32, tolerance


def make(lens, hq, hk, d, page, dtype, seed, dev, spare=3, width=None):
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width or max(max(need, default=0), 1)), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype).to(dev)
    kp, vp = (torch.randn(pages, hk, page, d, generator=g).to(dtype).to(dev) for _ in "kv")
    return q, kp, vp, table.to(dev)


def check(got, q, kp, vp, table, lens, **kw):
    o, mean, size = oracle.paged_attention(q, kp, vp, table.cpu(), lens, **kw)
    tol = tolerance(o, mean, size, q.dtype, max(lens), q.shape[2], float(vp.abs().max().float()))
    err = (got.double().cpu() - o).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (4, 4, 64), (16, 1, 128), (24, 1, 64), (40, 1, 128), (6, 2, 96)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_lengths(dev, hq, hk, d, page, dtype):
    from torchplusplus_amd.attention import paged_attention
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 129, 300, 513]
    q, kp, vp, table = make(lens, hq, hk, d, page, dtype, page, dev)
    check(paged_attention(q, kp, vp, table, i32(lens, dev)), q, kp, vp, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 128), (2, 2, 64), (2, 1, 256)])
@pytest.mark.parametrize("left", [0, 1, 15, 16, 100, 511, 2 ** 31 - 1, 2 ** 40])
def test_windows(dev, hq, hk, d, left):
    from torchplusplus_amd.attention import paged_attention
    lens = [1, 0, 33, 200, 700, 1025]
    q, kp, vp, table = make(lens, hq, hk, d, 32, torch.bfloat16, left % 97, dev)
    check(paged_attention(q, kp, vp, table, i32(lens, dev), window_left=left), q, kp, vp, table, lens, left=left)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 128, 1024])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_over_many_splits(dev, page, dtype):
    from torchplusplus_amd.attention import paged_attention
    lens = [9000, 40, 3001]
    q, kp, vp, table = make(lens, 8, 2, 128, page, dtype, 3, dev)
    check(paged_attention(q, kp, vp, table, i32(lens, dev)), q, kp, vp, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("b,hq,hk", [(70, 2, 1), (200, 4, 4), (600, 2, 2), (33, 32, 1)])
def test_many_sequences(dev, b, hq, hk):
    """Mixed lengths, some 0, more sequences than a wave has lanes, than are dealt splits."""
    from torchplusplus_amd.attention import paged_attention
    lens = [(i * i * 37) % 1400 if i % 7 else 0 for i in range(b)]
    lens[b // 2] = 3000
    q, kp, vp, table = make(lens, hq, hk, 64, 32, torch.bfloat16, b, dev)
    check(paged_attention(q, kp, vp, table, i32(lens, dev)), q, kp, vp, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 48])
def test_entries_that_are_no_page(dev, d):
    """Holes, entries past the pool and lengths past the table or below 0 read nothing."""
    from torchplusplus_amd.attention import paged_attention
    lens = [100, 64, 200, 17, 500, 90]
    q, kp, vp, table = make(lens, 4, 2, d, 16, torch.float16, 4, dev)
    pages = kp.shape[0]
    table[0, 2], table[0, 5] = -1, pages
    table[1, :] = -7                      # nothing left
    table[2, 0], table[2, 12] = 2 ** 31 - 1, -2 ** 31
    given = list(lens)
    given[3], given[4] = -5, 2 ** 31 - 1
    got = paged_attention(q, kp, vp, table, i32(given, dev))
    check(got, q, kp, vp, table, given)
    assert (got[1] == 0).all() and (got[3] == 0).all()
    none = paged_attention(q, kp[:0], vp[:0], table, i32(given, dev))
    assert (none == 0).all()
    assert (paged_attention(q, kp, vp, table[:, :0], i32(given, dev)) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 48])
def test_holes_behind_a_window(dev, d):
    """A row whose window shows holes alone is 0, whatever stands ahead of it; scores of
    -inf beside holes are NaN."""
    from torchplusplus_amd.attention import paged_attention
    lens = [200, 1000, 65, 1000]
    q, kp, vp, table = make(lens, 4, 2, d, 16, torch.float16, 11, dev)
    table[0, 11:], table[1, 60:], table[2, 4] = -1, -1, -1
    table[3, :30] = -1
    q[3] = q[3].abs() + 0.1
    for i in range(30, 63):
        kp[int(table[3, i])] = -math.inf
    for left in (0, 7, 20, 23):
        got = paged_attention(q, kp, vp, table, i32(lens, dev), window_left=left)
        o = oracle.paged_attention(q, kp, vp, table.cpu(), lens, left=left)[0]
        assert (got[:2] == 0).all() and torch.isnan(got[3]).all()
        assert (got[2].double().cpu() - o[2]).abs().max() < 0.01
    got = paged_attention(q, kp, vp, table, i32(lens, dev))
    assert torch.isnan(got[3]).all() and torch.isfinite(got[:3]).all()
    table[3, 30:] = -1
    assert (paged_attention(q, kp, vp, table, i32(lens, dev))[3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_that_are_not_seen_may_hold_anything(dev, d, dtype):
    from torchplusplus_amd.attention import paged_attention
    lens = [70, 1, 129, 16, 300]
    q, kp, vp, table = make(lens, 4, 2, d, 32, dtype, 5, dev)
    for i, x in enumerate((math.nan, math.inf, -math.inf, math.nan, math.inf)):
        page = int(table[i, lens[i] // 32]) if lens[i] % 32 else -1
        if page >= 0:
            kp[page, :, lens[i] % 32 :], vp[page, :, lens[i] % 32 :] = x, x
    check(paged_attention(q, kp.clone(), vp.clone(), table, i32(lens, dev)), q, kp.nan_to_num(0, 0, 0),
          vp.nan_to_num(0, 0, 0), table, lens)
    # in front of a window, and a page taken back
    first = int(table[4, 0])
    kp[first], vp[first] = math.nan, math.inf
    got = paged_attention(q, kp, vp, table, i32(lens, dev), window_left=250)
    table[4, 0] = -1
    check(got, q, kp.nan_to_num(0, 0, 0), vp.nan_to_num(0, 0, 0), table, lens, left=250)
    check(paged_attention(q, kp, vp, table, i32(lens, dev)), q, kp.nan_to_num(0, 0, 0), vp.nan_to_num(0, 0, 0), table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 48])
def test_values_that_are_not_finite_and_seen(dev, d):
    from torchplusplus_amd.attention import paged_attention
    lens = [300, 300, 300, 40]
    q, kp, vp, table = make(lens, 4, 2, d, 64, torch.bfloat16, 6, dev)
    vp[int(table[0, 1]), :, 5, 3] = math.inf
    vp[int(table[1, 2]), 1, 9, 0] = math.nan
    kp[int(table[2, 0])], kp[int(table[2, 1])] = -math.inf, -math.inf
    for i in (2, 3, 4):
        kp[int(table[2, i])] = -math.inf
    q[2] = q[2].abs() + 0.1
    got = paged_attention(q, kp, vp, table, i32(lens, dev))
    o = oracle.paged_attention(q, kp, vp, table.cpu(), lens)[0]
    assert torch.equal(torch.isnan(got).cpu(), torch.isnan(o)) and torch.equal(torch.isinf(got).cpu(), torch.isinf(o))
    assert (got[0, :, 3] == math.inf).all() and torch.isnan(got[2]).all() and torch.isfinite(got[3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 72])
def test_strides_scale_and_out(dev, d):
    """Keys and values interleaved in one pool, rows ahead of heads, a wide table's slice."""
    from torchplusplus_amd.attention import paged_attention
    lens = [130, 47, 1, 500]
    q, kp, vp, table = make(lens, 4, 2, d, 32, torch.float16, 7, dev)
    want = paged_attention(q, kp, vp, table, i32(lens, dev), softmax_scale=0.4)
    check(want, q, kp, vp, table, lens, scale=0.4)
    pool = torch.stack([kp, vp], 1).transpose(2, 3).contiguous().transpose(2, 3)  # [P, 2, rows, H, D] in memory
    wide = torch.full((4, 90), 1, dtype=torch.int32, device=dev)
    wide[:, 3 : 3 + table.shape[1]] = table
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.full((4, 9, d), 3.0, dtype=q.dtype, device=dev)[:, 2:6]
    got = paged_attention(qt, pool[:, 0], pool[:, 1], wide[:, 3 : 3 + table.shape[1]], i32(lens, dev), softmax_scale=0.4,
                          out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[700], [3000, 40, 2000, 1]])
def test_streams_and_graphs(dev, lens):
    """Side streams at once, and a captured call replayed with other lengths and tables,
    eager calls between the replays."""
    from torchplusplus_amd.attention import paged_attention
    q, kp, vp, table = make(lens, 16, 8, 128, 64, torch.bfloat16, 8, dev)
    n = i32(lens, dev)
    want = paged_attention(q, kp, vp, table, n)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(paged_attention(q, kp, vp, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, kp, vp, table, n)
        out2 = paged_attention(q, kp, vp, table, n)
    for step in range(4):
        n.copy_(i32([max(x - 13 * step, 0) for x in lens], dev))
        table[0, 0] = int(table[0, 1])
        want = paged_attention(q, kp, vp, table, n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want)


@pytest.mark.gpu
def test_refusals(dev):
    from torchplusplus_amd.attention import paged_attention
    lens = [20, 30]
    q, kp, vp, table = make(lens, 4, 2, 64, 16, torch.float16, 0, dev)
    n = i32(lens, dev)
    bad = torch.zeros(4, 2, 24, 64, dtype=torch.float16, device=dev)
    for args, kw in (((q.float(), kp, vp, table, n), {}), ((q, kp.bfloat16(), vp, table, n), {}),
                     ((q, kp, vp[1:], table, n), {}), ((q[:, :3], kp, vp, table, n), {}), ((q, bad, bad, table, n), {}),
                     ((q, kp[:, :, :8], vp[:, :, :8], table, n), {}), ((q, kp, vp, table.long(), n), {}),
                     ((q, kp, vp, table[:1], n), {}), ((q, kp, vp, table, n.long()), {}), ((q, kp, vp, table, n[:1]), {}),
                     ((q, kp, vp, table.cpu(), n), {}), ((q[:, None], kp, vp, table, n), {}), ((q, kp, vp, table, n), {"out": q}),
                     ((q, kp, vp, table, n), {"out": kp[0, :, :4].reshape(2, 4, 64)[:1]})):
        with pytest.raises(RuntimeError):
            paged_attention(*args, **kw)
