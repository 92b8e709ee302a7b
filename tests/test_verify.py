"""verify_draft against the 64-bit form in oracle/speculative.py: equal in
every output. Both sum in fp64 (by another order: 1e-16 of the sum apart, so a
uniform number of 24 bits meets a border between them at one draw in 10^7)."""
import pytest
import torch

from oracle import speculative as osp


def _probs(shape, gen, sharp=2.5, zeros=False):
    p = torch.softmax(torch.randn(shape, generator=gen) * sharp, -1)
    if zeros:
        p = p * (p >= p.amax(-1, keepdim=True) * 0.05)
        p = p / p.sum(-1, keepdim=True)
    return p


def _check(dev, tokens, p, u, q=None, parents=None):
    from torchplusplus_amd.llmops.speculative import verify_draft
    got = verify_draft(tokens.to(dev), p.to(dev), u.to(dev), None if q is None else q.to(dev),
                       None if parents is None else parents.to(dev))
    want = osp.verify_draft(tokens, p, u, q, parents)
    for g, w, n in zip(got, want, ("accepted", "path", "next_token")):
        assert g.dtype == w.dtype and torch.equal(g.cpu(), w), f"{n}: {g.cpu()} not {w}"
    return want


VOCABS = [1, 7, 100, 4096, 4097, 50257]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("b,t", [(1, 1), (5, 4), (3, 64)])
def test_chain_with_draft_probabilities(dev, dtype, vocab, b, t):
    g = torch.Generator().manual_seed(vocab + t)
    p = _probs((b, t + 1, vocab), g, zeros=vocab == 100)
    q = torch.softmax(torch.log(p[:, :t] + 1e-9) + 0.3 * torch.randn(b, t, vocab, generator=g), -1)
    tok = torch.multinomial(q.view(b * t, vocab), 1, generator=g).view(b, t)
    u = torch.rand(b, t + 1, generator=g)
    u[0] = 0.0  # accepts what has mass, draws the first index with mass
    _check(dev, tok, p.to(dtype), u, q.to(dtype))


def _tree(b, t, p, seed):
    g = torch.Generator().manual_seed(seed)
    par = torch.tensor([[int(torch.randint(max(-1, i - 5), i, (1,), generator=g)) for i in range(t)]
                        for _ in range(b)], dtype=torch.int32)
    best = p.argsort(-1, descending=True)
    tok = torch.zeros(b, t, dtype=torch.long)
    for i in range(b):
        met = {}
        for j in range(t):
            r = met.get(int(par[i, j]), 0)
            met[int(par[i, j])] = r + 1
            tok[i, j] = best[i, int(par[i, j]) + 1, min(r, p.shape[2] - 1)]
    return par, tok


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("b,t", [(1, 1), (6, 9), (2, 64)])
def test_tree_and_chain_of_chosen_tokens(dev, dtype, vocab, b, t):
    g = torch.Generator().manual_seed(vocab + 3 * t)
    p = _probs((b, t + 1, vocab), g, 3.5, zeros=vocab == 100).to(dtype)
    par, tok = _tree(b, t, p.float(), t)  # a small vocabulary gives siblings of one token
    for s in range(3):
        u = torch.rand(b, t + 1, generator=g)
        _check(dev, tok, p, u, None, par)
        _check(dev, tok, p, u)


@pytest.mark.gpu
def test_padding_and_rows_without_mass(dev):
    """Tokens outside the vocabulary, padded nodes, duplicate siblings, rows of
    zeros, NaN, infinities and negative masses, residuals without mass."""
    vocab, t, b = 60, 5, 6
    g = torch.Generator().manual_seed(7)
    p = _probs((b, t + 1, vocab), g, 1.0)
    q = _probs((b, t, vocab), g, 1.0)
    tok = torch.randint(0, vocab, (b, t), generator=g)
    u = torch.rand(b, t + 1, generator=g) * 0.3
    tok[0, 2], tok[1, 0], tok[2, 4] = -1, vocab, 10 ** 12
    p[3] = 0.0
    p[4, :, 1::2], p[4, :, 0], p[4, :, 2] = float("nan"), float("inf"), -1.0
    q[5, 0] = p[5, 0]      # nothing left of the target where it is refused
    u[5, 0] = 0.999999
    q[5, 0, tok[5, 0]], p[5, 0, tok[5, 0]] = 1.0, 0.0
    p[5, 0, :] = torch.where(torch.arange(vocab) == tok[5, 0], p[5, 0], torch.minimum(p[5, 0], q[5, 0]))
    want = _check(dev, tok, p, u, q)
    assert int(want[2][3]) == -1 and int(want[2][5]) >= 0 and int(want[0][1]) == 0
    par = torch.tensor([[-1, -1, 0, 0, 2], [-1, 7, 1, -2, 3], [-1, -1, -1, -1, -1], [-1, 0, 1, 2, 3],
                        [3, 4, -1, 2, 3], [-1, 0, 0, 0, 0]], dtype=torch.int32)
    tok[2] = 4             # five siblings of one token
    _check(dev, tok, p, u, None, par)
    one = torch.zeros(1, 2, vocab)
    one[0, :, 9] = 1.0     # all mass on the drafted token: always kept
    for x in (0.0, 0.5, 0.99999994):
        want = _check(dev, torch.tensor([[9]]), one, torch.tensor([[x, x]]))
        assert int(want[0]) == 1 and int(want[2]) == 9


@pytest.mark.gpu
def test_frequencies_follow_the_target(dev):
    """Tokens that come out are distributed as the target's first row, whatever
    was drafted: 20000 sequences, each bin within 5 standard deviations."""
    from torchplusplus_amd.llmops.speculative import verify_draft
    n, vocab = 20000, 6
    g = torch.Generator().manual_seed(11)
    p, q = _probs((2, vocab), g, 1.0), _probs((1, vocab), g, 1.0)
    for form in ("draft", "tree"):
        if form == "draft":
            tok = torch.multinomial(q.expand(n, -1), 1, generator=g)
            kw = dict(draft_probs=q.expand(n, 1, vocab).to(dev))
            pt = p.expand(n, 2, vocab)
        else:
            tok = torch.tensor([[2, 4, 2]]).expand(n, 3)
            kw = dict(parents=torch.full((n, 3), -1, dtype=torch.int32, device=dev))
            pt = p[[0, 1, 1, 1]].expand(n, 4, vocab)
        u = torch.rand(n, tok.shape[1] + 1, generator=g)
        acc, path, nxt = (x.cpu() for x in verify_draft(tok.to(dev), pt.to(dev), u.to(dev), **kw))
        first = torch.where(acc > 0, tok.gather(1, path[:, :1].clamp(min=0).long())[:, 0], nxt)
        share = torch.bincount(first, minlength=vocab) / n
        assert bool(((share - p[0]).abs() <= 5 * (p[0] / n).sqrt()).all()), f"{form}: {share} not {p[0]}"


@pytest.mark.gpu
def test_captured_strided_and_repeated(dev):
    """Rows with gaps between them, a captured call replayed on new numbers, the
    same call twice."""
    from torchplusplus_amd.llmops.speculative import verify_draft
    b, t, vocab = 3, 4, 9001
    g = torch.Generator().manual_seed(5)
    p, q = _probs((b, t + 1, vocab), g), _probs((b, t, vocab), g)
    tok = torch.multinomial(q.view(-1, vocab), 1, generator=g).view(b, t)
    wide = torch.full((b, t + 2, vocab + 3), float("nan"), device=dev)
    wide[:, : t + 1, :vocab] = p.to(dev)
    ps, qd, td = wide[:, : t + 1, :vocab], q.to(dev), tok.to(dev)
    ud = torch.rand(b, t + 1, generator=g).to(dev)
    verify_draft(td, ps, ud, qd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_draft(td, ps, ud, qd)
    for _ in range(4):
        u = torch.rand(b, t + 1, generator=g)
        ud.copy_(u)
        graph.replay()
        eager = verify_draft(td, ps, ud, qd)
        want = osp.verify_draft(tok, p, u, q)
        assert all(torch.equal(a.cpu(), w) and torch.equal(e.cpu(), w) for a, e, w in zip(got, eager, want))


def test_refuses_cpu_tensors():
    from torchplusplus_amd.llmops.speculative import verify_draft
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_draft(torch.zeros(1, 1, dtype=torch.long), torch.ones(1, 2, 4), torch.zeros(1, 2))


@pytest.mark.gpu
def test_refusals(dev):
    from torchplusplus_amd.llmops.speculative import verify_draft
    tok, p = torch.zeros(2, 3, dtype=torch.long, device=dev), torch.ones(2, 4, 10, device=dev)
    u, par = torch.zeros(2, 4, device=dev), torch.full((2, 3), -1, dtype=torch.int32, device=dev)
    for args in ((tok.int(), p, u), (tok[:1], p, u), (tok, p[:, :3], u), (tok, p.double(), u), (tok, p, u[:, :3]),
                 (tok, p, u.double()), (tok, p, u, p), (tok, p, u, p[:, :3].half()), (tok, p, u, None, par.long()),
                 (tok, p, u, None, par[:, :2]), (tok, p, u, p[:, :3], par), (tok.cpu(), p, u),
                 (tok, p[..., :0], u), (tok, p.transpose(1, 2)[:, :4, :], u), (tok[:, :0], p[:, :1], u[:, :1]),
                 (torch.zeros(1, 65, dtype=torch.long, device=dev), torch.ones(1, 66, 4, device=dev),
                  torch.zeros(1, 66, device=dev))):
        with pytest.raises(RuntimeError):
            verify_draft(*args)
    assert verify_draft(tok[:0], p[:0], u[:0])[1].shape == (0, 3)
