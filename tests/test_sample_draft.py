"""LLMInference.sample_draft at the ends of the temperature's range."""
import math

import pytest
import torch

from oracle import speculative as osp


def test_refuses_a_temperature_below_0():
    from tests.test_llmops import TinyLM
    for temp in (-1.0, math.nan):
        with pytest.raises(ValueError, match="temp"):
            TinyLM().sample_draft(torch.zeros(1, 2, dtype=torch.long), torch.zeros(1, 3, 9), temp)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperature_0_is_greedy(dev, dtype):
    """The drafted tokens that greedy decoding would give stay, whatever the uniform
    numbers, and the next is the largest logit's, for a chain and a tree."""
    from tests.test_llmops import TinyLM
    g = torch.Generator().manual_seed(3)
    b, t, v = 3, 4, 40
    logits = -torch.randint(0, 9, (b, t + 1, v), generator=g).to(dtype)
    best = torch.randint(0, v, (b, t + 1), generator=g)
    logits.scatter_(-1, best.unsqueeze(-1), 0.5)  # no ties
    tok = best[:, :t].clone()
    tok[1, 2] = (tok[1, 2] + 1) % v
    n, path, nxt = TinyLM().sample_draft(tok.to(dev), logits.to(dev), 0.0)
    assert n.tolist() == [4, 2, 4] and nxt.tolist() == [int(best[0, 4]), int(best[1, 2]), int(best[2, 4])]
    q = torch.softmax(torch.randn(b, t, v, generator=g), -1)
    got = TinyLM().sample_draft(tok.to(dev), logits.to(dev), 0, draft_probs=q.to(dev))
    assert got[0].tolist() == [4, 2, 4] and got[2].tolist() == nxt.tolist()
    par = torch.tensor([[-1, -1, 1, 2]] * b, dtype=torch.int32)
    tree = torch.stack([(best[:, 0] + 1) % v, best[:, 0], best[:, 2], best[:, 3]], 1)  # all but the first stay
    n, path, nxt = TinyLM().sample_draft(tree.to(dev), logits.to(dev), 0.0, parents=par.to(dev))
    u = torch.rand(b, t + 1, generator=g)
    one = torch.nn.functional.one_hot(best, v).float()
    want = osp.verify_draft(tree, one, u, None, par)
    assert path.tolist() == [[1, 2, 3, -1]] * b and nxt.tolist() == best[:, 4].tolist()
    assert torch.equal(n.cpu(), want[0]) and torch.equal(nxt.cpu(), want[2])
