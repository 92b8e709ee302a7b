"""Tensors that share memory: what a call would write twice, or write where it reads,
is refused before anything is launched; layouts that only interleave are not."""
import pytest
import torch


@pytest.mark.gpu
def test_rotation_in_place(dev):
    from torchplusplus_amd.dlops.rope import rope_apply_at, rope_apply_at_
    b, s, h, d = 2, 3, 4, 64
    p, f = torch.arange(s, device=dev).int(), torch.ones(d // 2, dtype=torch.float64, device=dev)
    x = torch.randn(1 << 14, device=dev).half()
    view = lambda off, st, n=h: x.as_strided((b, s, n, d), (*st, 1), off)  # noqa: E731
    before = x.clone()
    for q, k in ((view(0, (d, d, 8 * d)), None),                 # (1, 0) is (0, 1)
                 (view(0, (s * 2 * d, 2 * d, d)), None),         # heads reach into the next token
                 (view(0, (s * 4 * d, 4 * d, d // 2)), None),
                 (view(0, (3000, 1000, d)), view(d // 2, (3000, 1000, d))),      # half a head on
                 (view(0, (3000, 1000, d)), view(2 * d, (3000, 1000, d), 2)),    # two heads of q
                 (view(0, (3000, 1000, d)), view(1000, (3000, 1000, d), 2)),     # the next token's
                 (view(0, (3000, 1000, d)), view(64, (4000, 1300, 200), 2))):
        with pytest.raises(RuntimeError, match="overlap"):
            rope_apply_at_(q, k, p, f)
    assert torch.equal(x, before)
    # a fused projection, heads of q and k in turn, k behind q, another order of dims
    for q, k in ((view(0, (3000, 1000, d)), view(4 * d, (3000, 1000, d), 2)),
                 (view(0, (3000, 1000, 2 * d)), view(d, (3000, 1000, 2 * d))),
                 (view(0, (s * h * d, h * d, d)), view(b * s * h * d, (s * h * d, h * d, d))),
                 (view(0, (h * s * d, d, s * d)), None), (view(0, (d, b * d, b * s * d)), None)):
        want = rope_apply_at(q, k, p, f)
        got = rope_apply_at_(q, k, p, f)
        assert torch.equal(got[0], want[0]) and (k is None or torch.equal(got[1], want[1]))


@pytest.mark.gpu
def test_append(dev):
    from torchplusplus_amd.llmops.kvcache import kv_quant_append, kv_quant_read
    b, s, h, d, room = 2, 3, 2, 64, 16
    k, v = (torch.randn(b, s, h, d, device=dev).half() for _ in "kv")
    codes = torch.zeros(1 << 16, dtype=torch.int8, device=dev)
    exps = torch.full((1 << 12,), 127, dtype=torch.uint8, device=dev)
    n = h * room * d
    c = lambda off, st=(n, room * d): codes.as_strided((b, h, room, d), (*st, d, 1), off)  # noqa: E731
    e = lambda off, st=(h * room, room): exps.as_strided((b, h, room), (*st, 1), off)  # noqa: E731
    pos = torch.zeros(b, dtype=torch.int32, device=dev)
    for bad in ((c(0), c(n), e(0), e(1000)),                                # V's first sequence is K's second
                (c(0), c(room * d), e(0), e(1000)),                         # one head on
                (c(0), c(2 * n - 8), e(0), e(1000)),
                (c(0), c(2 * n), e(0), e(h * room)),
                (c(0, (d, room * d)), c(20000, (d, room * d)), e(0), e(1000)),  # sequences a row apart
                (c(0), c(2 * n), e(0, (4, room)), e(1000, (4, room))),
                (c(0), c(2 * n), codes.view(torch.uint8)[64 : 64 + b * h * room].view(b, h, room), e(0))):
        with pytest.raises(RuntimeError, match="of their own"):
            kv_quant_append(k, v, *bad, pos)
    inside = codes.view(torch.float16)[: b * s * h * d].view(b, s, h, d)
    for kk, vv in ((inside, v), (k, inside)):
        with pytest.raises(RuntimeError, match="in the cache"):
            kv_quant_append(kk, vv, c(0), c(2 * n), e(0), e(1000), pos)
    assert not bool(codes.any())
    # K and V of a sequence, or of a head, in turn
    for kc, vc in ((c(0, (2 * n, room * d)), c(n, (2 * n, room * d))),
                   (c(0, (2 * n, 2 * room * d)), c(room * d, (2 * n, 2 * room * d))),
                   (c(0, (room * d, b * room * d)), c(2 * n, (room * d, b * room * d)))):
        kv_quant_append(k, v, kc, vc, e(0), e(1000), pos)
        ref = [torch.zeros(b, h, room, d, dtype=torch.int8, device=dev) for _ in "kv"]
        kv_quant_append(k, v, *ref, e(0), e(1000), pos)
        assert torch.equal(kc[:, :, :s], ref[0][:, :, :s]) and torch.equal(vc[:, :, :s], ref[1][:, :, :s])
        got = kv_quant_read(kc, vc, e(0), e(1000), s)
        assert float((got[0].transpose(1, 2).float() - k.float()).abs().max()) <= 0.0625  # half a step up to 8


@pytest.mark.gpu
def test_attention_output(dev):
    from torchplusplus_amd.attention import tree_attention
    b, t, h, d, room = 2, 3, 4, 64, 32
    n, par = torch.full((b,), 5, dtype=torch.int32, device=dev), torch.full((b, t), -1, dtype=torch.int32, device=dev)
    q = torch.randn(b, t, h, d, device=dev).half()
    kc, vc = (torch.randint(-9, 9, (b, h, room, d), device=dev, dtype=torch.int8) for _ in "kv")
    size = b * t * h * d
    for which in range(4):  # the output over exponents, lengths, parents; over itself
        mem = torch.zeros(2 * size, dtype=torch.uint8, device=dev)
        o = mem.view(torch.float16).view(b, t, h, d)
        e = [torch.full((b, h, room), 120, dtype=torch.uint8, device=dev) for _ in "kv"]
        lens, parents = n, par
        if which == 0:
            e[1] = mem[2 * size - b * h * room :].view(b, h, room).fill_(120)
        elif which == 1:
            lens = mem[:8].view(torch.int32).fill_(5)
        elif which == 2:
            parents = mem[64 : 64 + 4 * b * t].view(torch.int32).view(b, t).fill_(-1)
        else:
            o = torch.zeros(4096, dtype=torch.float16, device=dev).as_strided((b, t, h, d), (d, d, 8 * d, 1))
        with pytest.raises(RuntimeError, match="of its own"):
            tree_attention(q, kc, vc, lens, parents, k_exps=e[0], v_exps=e[1], out=o)
    both = torch.randn(b, t, h, 2 * d, device=dev).half()  # query and output in turn
    want = tree_attention(both[..., :d], kc, vc, n, par, k_exps=e[0], v_exps=e[1])
    got = tree_attention(both[..., :d], kc, vc, n, par, k_exps=e[0], v_exps=e[1], out=both[..., d:])
    assert torch.equal(got, want) and got.data_ptr() == both[..., d:].data_ptr()
