"""PagedKVCache where a step is empty, or is not one (CPU)."""
import pytest
import torch

from tests.test_paged_cache import cache
from torchplusplus_amd.llmops.paged import PagedKVCache


def test_table_of_no_pages():
    c = cache()
    seqs = [c.allocate(), c.allocate()]
    step = c.decode_step(c.block_tables(seqs), torch.tensor([0, 5], dtype=torch.int32))
    assert step.slots.dtype == torch.int64 and step.slots.tolist() == [-1, -1]
    assert c.decode_step(c.block_tables([]), torch.zeros(0, dtype=torch.int32)).slots.shape == (0,)


@pytest.mark.parametrize("starts,counts", [([0], [3, 4]), ([0, 0], [3]), ([0, 0, 0], [3, 4, 5])])
def test_lists_of_other_lengths(starts, counts):
    c = cache()
    seqs = [c.allocate(16), c.allocate(16)]
    for call in (c.slots, c.prefill_step):
        with pytest.raises(ValueError, match="one start and one count"):
            call(seqs, starts, counts)


@pytest.mark.parametrize("starts,counts", [([0, -1], [40, 1]), ([0, 4], [40, -1]), ([-30, 0], [1, 40])])
def test_refused_step_deals_nothing(starts, counts):
    c = cache()
    seqs = [c.allocate(), c.allocate()]
    with pytest.raises(ValueError):
        c.prefill_step(seqs, starts, counts)
    assert c.free_pages == 6 and c.pages_of(seqs[0]) == []


def test_empty_step():
    c = cache()
    s = c.prefill_step([], [], [])
    assert s.cu_seqlens.tolist() == [0] and s.slots.shape == (0,) and s.positions.shape == (0,)
    a = c.allocate(5)
    s = c.prefill_step([a], [5], [0])
    assert s.cu_seqlens.tolist() == [0, 0] and s.cu_seqlens_k.tolist() == [0, 5] and len(s.key_slots) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 40])
def test_model_of_empty_and_padded_steps(dev, n):
    """No tokens, no rows wanted, a decode batch padded by a sequence at position -1 without
    pages: logits of the shapes asked for, and nothing written outside a sequence's pages."""
    from tests.test_model import TINY16 as cfg
    from torchplusplus_amd.fastqwen3 import FastQwen3
    with torch.inference_mode():
        m = FastQwen3(cfg, device=dev).eval()
        m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(1))
        c = PagedKVCache(6, 16, cfg.n_layers, cfg.n_kv_heads, cfg.head_dim, cfg.dtype, dev)
        none = torch.zeros(0, dtype=torch.int64, device=dev)
        assert m.forward_paged(none, c, c.prefill_step([], [], [])).shape == (0, cfg.vocab_size)
        a, b = c.allocate(n + 1), c.allocate()
        ids = torch.arange(n, device=dev) % cfg.vocab_size
        assert m.forward_paged(ids, c, c.prefill_step([a], [0], [n]), none).shape == (0, cfg.vocab_size)
        k, v = c.read(1, c.slots([a], [0], [n])[1])
        assert (k != 0).any(2).all() and (v != 0).any(2).all()  # written all the same
        step = c.decode_step(c.block_tables([a, b]), torch.tensor([n, -1], dtype=torch.int32, device=dev))
        assert step.slots.tolist()[1] == -1 and step.seqlens.tolist() == [n + 1, 0]
        assert m.forward_paged(ids[:2], c, step).isfinite().all()
        m.check_device_errors()
        others = [x for x in range(6) if x not in c.pages_of(a)]
        assert (c.k_pages[:, others] == 0).all() and (c.v_pages[:, others] == 0).all()
