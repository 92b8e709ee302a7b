"""LLMInference.score takes token ids of the types that a forward pass does."""
import pytest
import torch


@pytest.mark.gpu
def test_int32_ids(dev):
    from tests.test_model import TINY16 as cfg
    from torchplusplus_amd.fastqwen3 import FastQwen3
    with torch.inference_mode():
        m = FastQwen3(cfg, device=dev).eval()
        m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(1))
        ids = torch.randint(0, cfg.vocab_size, (2, 9), generator=torch.Generator().manual_seed(2)).to(dev)
        assert torch.equal(m.forward(ids.int()), m.forward(ids))
        assert all(torch.equal(a, b) for a, b in zip(m.score(ids.int(), 3), m.score(ids, 3)))
