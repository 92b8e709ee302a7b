"""Rows further than 2^32 bytes and 2^31 elements from a tensor's start: results must be bit
for bit those of a compact copy."""
import pytest
import torch

FAR = 2 ** 31 + 2 ** 20  # elements


def spread(x):
    """x with dim 0 spread over FAR elements (the gaps are not initialised)."""
    step = (FAR // (x.shape[0] - 1)) // 8 * 8
    store = torch.empty(step * (x.shape[0] - 1) + x[0].numel(), dtype=x.dtype, device=x.device)
    far = store.as_strided(x.shape, (step, *x.stride()[1:]))
    return far.copy_(x)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("lens", [[3, 150], [700, 90], [700] * 100])
def test_packed(dev, d, lens):
    from torchplusplus_amd.attention import packed_attention
    g = torch.Generator().manual_seed(1)
    n = sum(lens)
    q, k, v = (torch.randn(n, h, d, generator=g).bfloat16().to(dev) for h in (4, 2, 2))
    cu = torch.tensor([0, *lens]).cumsum(0).int().to(dev)
    want = packed_attention(q, k, v, cu)
    out = spread(torch.zeros_like(q))
    got = packed_attention(spread(q), spread(k), spread(v), cu, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("left", [-1, 90])
def test_paged_and_rope(dev, d, left):
    from torchplusplus_amd.attention import paged_attention
    from torchplusplus_amd.llmops.paged import qkv_rope_paged
    g = torch.Generator().manual_seed(2)
    hq, hk, page = 8, 2, 32
    kp, vp = (torch.randn(20, hk, page, d, generator=g).half().to(dev) for _ in "kv")
    far_k, far_v = spread(kp), spread(vp)
    if d != 48:
        cos, sin = (torch.randn(64, d, generator=g).to(dev) for _ in "cs")
        qkv = torch.randn(20, (hq + 2 * hk) * d, generator=g).half().to(dev)
        pos = torch.arange(20, dtype=torch.int32, device=dev)
        slots = (torch.arange(20, device=dev) * page + 31 - pos).long()  # a row of every page
        a = qkv_rope_paged(qkv, pos, slots, kp, vp, cos, sin)
        b = qkv_rope_paged(qkv, pos, slots, far_k, far_v, cos, sin)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert torch.equal(kp, far_k) and torch.equal(vp, far_v)
    q = torch.randn(3, hq, d, generator=g).half().to(dev)
    table = torch.randperm(20, generator=g)[:18].int().view(3, 6).to(dev)
    lens = torch.tensor([192, 1, 130], dtype=torch.int32, device=dev)
    want = paged_attention(q, kp, vp, table, lens, window_left=left)
    assert torch.equal(paged_attention(q, far_k, far_v, table, lens, window_left=left), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1000, 40001])
def test_logprobs(dev, dtype, v):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    g = torch.Generator().manual_seed(3)
    x = (3 * torch.randn(4, v, generator=g)).to(dtype).to(dev)
    tokens = torch.randint(0, v, (4,), generator=g).to(dev)
    for a, b in zip(token_logprobs(x, tokens, 7), token_logprobs(spread(x), tokens, 7)):
        assert torch.equal(a, b)
