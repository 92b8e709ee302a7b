"""Rows whose largest logits stand in fewer places than alternatives are asked for: all of the
row's elements of `top` - 1 of 64 places, a place being eight neighbours in every 512, are raised
above the others. 4 (top - 1) runs of eight in every 2048 elements are then above the top-th
place's maximum, up to 993 a block, over a thousand elements. Tolerances: test_token_logprobs.py."""
import pytest
import torch

from tests.test_token_logprobs import check

KINDS = 3


def raised(v, top, dtype, seed, shift=0):
    """KINDS rows: noise, raised by 10, 10 + 5 i / v and 10 at places shift, shift + 1, ..."""
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(v)
    up = ((i // 8 - shift) % 64 < top - 1).float()
    noise = torch.randn(KINDS, v, generator=g)
    return torch.stack([noise[0] + 10 * up, noise[1] + (10 + 5 * i / v) * up, noise[2].clamp(max=0.5) + 10 * up]).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [9, 20, 32])
@pytest.mark.parametrize("n,v", [(300, 16384), (700, 6144), (300, 16385), (8, 151936), (100, 32768), (40, 50257), (600, 20000)])
def test_largest_in_few_places(dev, n, v, top, dtype):
    """Whole rows and chunks of them, of up to eight iterations a block and more."""
    from torchplusplus_amd.llmops.scoring import token_logprobs
    for shift in (0, 41):
        x = raised(v, top, dtype, v + top, shift).to(dev)
        at = (torch.arange(n) % KINDS).to(dev)
        t = torch.arange(n, device=dev) * 1237 % v
        r, again = (token_logprobs(x[at], t, top) for _ in range(2))
        assert all(torch.equal(a, b) for a, b in zip(r, again))
        few = slice(0, min(n, KINDS))  # (the rest are the same rows)
        check(type(r)(*(y[few] for y in r)), x[at[few]], t[few], top)
        for k in range(min(n, KINDS)):
            assert (r.top_tokens[at == k] == r.top_tokens[k]).all() and (r.top_logprobs[at == k] == r.top_logprobs[k]).all()
