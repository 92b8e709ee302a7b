"""A decode step of FastQwen3 over pages as a HIP graph: every replay, with eager work of the
same operators in between, against an eager run over a cache of its own."""
import pytest
import torch

from tests.test_model import TINY16 as cfg


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[40, 3], [130, 1, 64, 17]])
def test_captured_decode(dev, lens):
    from torchplusplus_amd.fastqwen3 import FastQwen3
    from torchplusplus_amd.llmops.paged import PagedKVCache
    from torchplusplus_amd.llmops.scoring import token_logprobs
    steps = 6
    with torch.inference_mode():
        m = FastQwen3(cfg, device=dev).eval()
        m.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(1))
        g = torch.Generator().manual_seed(2)
        ids = torch.cat([torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in lens]).to(dev)

        class Run:
            def __init__(self):
                self.cache = PagedKVCache(24, 16, cfg.n_layers, cfg.n_kv_heads, cfg.head_dim, cfg.dtype, dev)
                seqs = [self.cache.allocate(n + steps + 1) for n in lens]
                step = self.cache.prefill_step(seqs, [0] * len(lens), lens)
                logits = m.forward_paged(ids, self.cache, step, step.cu_seqlens[1:].long() - 1)
                self.table = self.cache.block_tables(seqs)
                self.pos = torch.tensor(lens, dtype=torch.int32, device=dev)
                self.tokens = logits.argmax(1)

            def step(self):
                logits = m.forward_paged(self.tokens, self.cache, self.cache.decode_step(self.table, self.pos))
                self.pos.add_(1)
                self.tokens.copy_(logits.argmax(1))
                return logits, token_logprobs(logits, self.tokens, 3)

        eager, captured = Run(), Run()
        assert torch.equal(eager.tokens, captured.tokens)
        pos, tokens = captured.pos.clone(), captured.tokens.clone()
        captured.step()  # warm: written over by the first replay
        captured.pos.copy_(pos), captured.tokens.copy_(tokens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = captured.step()
        captured.pos.copy_(pos), captured.tokens.copy_(tokens)
        for i in range(steps):
            logits, scores = eager.step()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], logits), i
            assert all(torch.equal(a, b) for a, b in zip(out[1], scores)), i
            assert torch.equal(captured.tokens, eager.tokens) and torch.equal(captured.pos, eager.pos), i
        m.check_device_errors()
