"""A serving loop over FastQwen3 with a paged cache: prompts together, sequences that end and
give their pages to others, a follow-up turn. Tokens must be the largest logits' of a forward
pass over each sequence's own history, within the pass's rounding (as test_serving_step.py)."""
import pytest
import torch

from tests.test_model import TINY16 as cfg


@pytest.mark.gpu
def test_loop(dev):
    from torchplusplus_amd.fastqwen3 import FastQwen3
    from torchplusplus_amd.llmops.paged import PagedKVCache
    from torchplusplus_amd.llmops.scoring import token_logprobs
    with torch.inference_mode():
        model = FastQwen3(cfg, device=dev).eval()
        model.init_weights(std=0.05, generator=torch.Generator(device=dev).manual_seed(1))
        g = torch.Generator().manual_seed(2)
        new = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).to(dev)  # noqa: E731
        cache = PagedKVCache(12, 16, model.get_num_layers(), model.get_kv_heads(), model.get_head_dim(), model.get_dtype(), dev)
        history = {}

        def prefill(seqs, texts):
            lens = [len(history[s]) if s in history else 0 for s in seqs]
            step = cache.prefill_step(seqs, lens, [len(t) for t in texts])
            logits = model.forward_paged(torch.cat(texts), cache, step, step.cu_seqlens[1:].long() - 1)
            for s, t in zip(seqs, texts):
                history[s] = torch.cat([history[s], t]) if s in history else t
            return logits.argmax(-1)

        def decode(seqs, tokens, steps):
            positions = torch.tensor([len(history[s]) for s in seqs], dtype=torch.int32, device=dev)
            for _ in range(steps):
                for s, t in zip(seqs, tokens):
                    cache.grow(s, len(history[s]) + 1)
                    history[s] = torch.cat([history[s], t.view(1)])
                logits = model.forward_paged(tokens, cache, cache.decode_step(cache.block_tables(seqs), positions))
                tokens, positions = logits.argmax(-1), positions + 1
                scores = token_logprobs(logits, tokens, top_k=3)
                assert torch.equal(scores.top_tokens[:, 0], tokens)
                for i, s in enumerate(seqs):  # against the sequence's history on its own
                    own = model.forward(history[s].view(1, -1))[0, -1].float()
                    assert own.amax() - own[tokens[i]] <= 0.05
                    assert (scores.logprobs[i] - own.log_softmax(0)[tokens[i]]).abs() < 0.06
            return tokens

        a, b = cache.allocate(), cache.allocate()
        tokens = decode([a, b], prefill([a, b], [new(33), new(2)]), 4)
        cache.free(b)
        c = cache.allocate()
        first = prefill([c], [new(60)])
        decode([c, a], torch.stack([first[0], tokens[0]]), 5)
        turn = prefill([a], [new(7)])  # a's last token is not cached: its turn begins behind the cached ones
        decode([a, c], torch.stack([turn[0], new(1)[0]]), 3)
        model.check_device_errors()
