"""Whole rows and chunks of them, short enough to stay in registers and longer, on rows whose
equal logits fill the list of candidates."""
import pytest
import torch

from tests.test_token_logprobs import check


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(700, 9001), (300, 33000), (20, 400003), (200, 60001), (5, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties(dev, n, v, dtype):
    from torchplusplus_amd.llmops.scoring import token_logprobs
    i = torch.arange(v, dtype=torch.float32)
    g = torch.Generator().manual_seed(v)
    noise = torch.randn(v, generator=g)
    kinds = [torch.zeros(v), i % 7, (i % 2048 < 8) * 20.0, (i % 2048 < 256) * 30.0 + noise.clamp(max=0), noise.round(),
             torch.where(i < v - 3, float("-inf"), 1.0), (i % 4096 == 4095) * 3.0, noise.clamp(max=0.5), i / v, -i / v]
    x = torch.stack([kinds[r % len(kinds)] for r in range(len(kinds))]).to(dtype).to(dev)
    at = torch.arange(n) % len(kinds)
    t = torch.arange(n, device=dev) * 1237 % v
    for top in (1, 17, 32):
        r = token_logprobs(x[at.to(dev)], t, top)
        few = torch.arange(min(n, 2 * len(kinds)))  # (the rest are the same rows)
        check(type(r)(*(y[few.to(dev)] for y in r)), x[at[few].to(dev)], t[few.to(dev)], top)
        for k in range(len(kinds)):
            same = (at == k).nonzero().squeeze(1).to(dev)
            assert (r.top_tokens[same] == r.top_tokens[same[:1]]).all() and (r.entropy[same] == r.entropy[same[:1]]).logical_or(
                r.entropy[same].isnan()).all()
