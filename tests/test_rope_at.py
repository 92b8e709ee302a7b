"""rope_apply_at against the 64-bit form in oracle/speculative.py.

Tolerance of an element: its own rounding to T, eps / 2 of it (and half the
least fp16 step, 2^-25), and the fp32 rotation: cos and sin to 2e-7 (hardware
to 1.3e-7, the angle rounded to 2^-25 turns, 2 pi of which is 1.9e-7 at most;
together below 4e-7), times factor, two products and a sum (3 * 2^-24), all of
the sum of the two terms' sizes: 6e-7 of it."""
import math

import pytest
import torch

from oracle import speculative as osp

THETA = 1e6
# B, S, Hq, Hk, D, R: one token; odd counts; part of a head; sizes that take
# every width of access (8, 4, 2, 1 pairs)
SHAPES = [(1, 1, 1, 1, 64, 64), (2, 5, 16, 8, 128, 128), (1, 17, 3, 1, 80, 80), (3, 2, 4, 2, 64, 20),
          (1, 33, 2, 2, 128, 64), (2, 3, 5, 5, 256, 256), (1, 4, 2, 1, 72, 24), (1, 3, 2, 1, 10, 6),
          (1, 3, 3, 0, 128, 32), (1, 2, 1, 1, 2, 2)]


def _close(got, exact, terms, what):
    got, eps = got.double().cpu(), torch.finfo(got.dtype).eps
    tol = eps / 2 * exact.abs() * (1 + eps) + 2.0 ** -25 + 6e-7 * terms
    bad = (got - exact).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, by up to {float((got - exact).abs().max())}"


def _case(shape, dtype, seed, far):
    b, s, hq, hk, d, r = shape
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, s, (hq + 2 * hk) * d, generator=g).to(dtype)
    pos = torch.randint(0, far, (b, s), generator=g, dtype=torch.int32)
    f = THETA ** (-2.0 * torch.arange(r // 2, dtype=torch.float64) / r)
    return qkv, pos, f


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rope_at(dev, dtype, interleaved, shape):
    """Views of a fused projection, far positions, padding tokens, a factor."""
    from torchplusplus_amd.dlops.rope import rope_apply_at
    b, s, hq, hk, d, r = shape
    qkv, pos, f = _case(shape, dtype, 1 + s, 1000000)
    pos[0, s // 2] = -1
    x = qkv.to(dev)
    q = x[..., : hq * d].view(b, s, hq, d)
    k = x[..., hq * d : (hq + hk) * d].view(b, s, hk, d) if hk else None
    got = rope_apply_at(q, k, pos.to(dev), f.to(dev), interleaved, 1.25)
    for n, g in zip((q, k), got):
        if n is not None:
            exact, terms = osp.rope_at(n.cpu(), pos, f, interleaved, 1.25)
            _close(g, exact, terms, f"rope_at {shape}")
    assert got[0].is_contiguous() and torch.equal(got[0][0, s // 2], q[0, s // 2])
    assert torch.equal(x.cpu(), qkv), "the input was written"


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_at_in_place(dev, interleaved):
    """In place on views of a fused projection equals out of place, and leaves
    the values between them alone; int64 and shared positions."""
    from torchplusplus_amd.dlops.rope import rope_apply_at, rope_apply_at_
    b, s, hq, hk, d = 2, 7, 4, 2, 128
    qkv, _, f = _case((b, s, hq, hk, d, 64), torch.bfloat16, 5, 10)
    pos = torch.arange(3, 3 + s)
    x = qkv.to(dev)
    views = lambda t: (t[..., : hq * d].view(b, s, hq, d), t[..., hq * d : (hq + hk) * d].view(b, s, hk, d))  # noqa: E731
    q, k = views(x)
    want = rope_apply_at(q, k, pos.to(dev).int().expand(b, s).contiguous(), f.to(dev), interleaved)
    got = rope_apply_at_(q, k, pos.to(dev), f.to(dev), interleaved)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert got[0].data_ptr() == x.data_ptr()
    assert torch.equal(x[..., (hq + hk) * d :].cpu(), qkv[..., (hq + hk) * d :])


@pytest.mark.gpu
def test_rope_at_is_the_table_form(dev):
    """At positions 0 .. S - 1 and with the plain frequencies: qkrope_apply on
    fp32 tables. Both round once, from fp32 results 1e-6 of the terms apart, so
    at most one bit differs."""
    from torchplusplus_amd.dlops.rope import (compute_rope_params, qkrope_apply, rope_apply_at,
                                              rope_frequencies)
    q, k = torch.randn(2, 50, 4, 64, device=dev).bfloat16(), torch.randn(2, 50, 2, 64, device=dev).bfloat16()
    cos, sin = compute_rope_params(64, THETA, 50, device=dev, dtype=torch.float64, out_dtype=torch.float32)
    tq, tk = qkrope_apply(q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), cos, sin)
    f, factor = rope_frequencies(64, THETA, device=dev)
    gq, gk = rope_apply_at(q, k, torch.arange(50, device=dev), f, attention_factor=factor)
    for g, t in ((gq, tq), (gk, tk)):
        diff = (g.float() - t.transpose(1, 2).float()).abs()
        assert bool((diff <= torch.finfo(torch.bfloat16).eps * t.transpose(1, 2).float().abs() + 1e-5).all())


@pytest.mark.gpu
def test_rope_at_captured_and_on_a_stream(dev):
    from torchplusplus_amd.dlops.rope import rope_apply_at
    qkv, pos, f = _case((2, 9, 4, 4, 64, 64), torch.float16, 2, 5000)
    q = qkv.to(dev)[..., : 4 * 64].view(2, 9, 4, 64)
    p, fd = pos.to(dev), f.to(dev)
    want = rope_apply_at(q, q, p, fd)[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert torch.equal(rope_apply_at(q, None, p, fd)[0], want)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = rope_apply_at(q, None, p, fd)[0]
    for _ in range(3):
        o.zero_()
        graph.replay()
        assert torch.equal(o, want)


def test_frequencies():
    from torchplusplus_amd.dlops.rope import rope_frequencies
    f, a = rope_frequencies(128, THETA, device="cpu")
    assert f.dtype == torch.float64 and len(f) == 64 and f[0] == 1 and a == 1
    assert abs(float(f[1]) - THETA ** (-2 / 128)) < 1e-15
    lin, a = rope_frequencies(128, THETA, "linear", 4.0, device="cpu")
    assert torch.equal(lin, f / 4) and a == 1
    ntk, a = rope_frequencies(128, THETA, "ntk", 4.0, device="cpu")
    assert ntk[0] == 1 and abs(float(ntk[-1] / f[-1]) - 0.25) < 1e-12 and a == 1
    yarn, a = rope_frequencies(128, 1e4, "yarn", 4.0, original_context=4096, device="cpu")
    base, _ = rope_frequencies(128, 1e4, device="cpu")
    turns = 4096 * base / (2 * math.pi)
    assert torch.equal(yarn[turns > 34], base[turns > 34])
    assert torch.allclose(yarn[turns < 0.9], base[turns < 0.9] / 4, rtol=1e-15)
    assert bool((yarn[1:] < yarn[:-1]).all()) and abs(a - (0.1 * math.log(4) + 1)) < 1e-15
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, scaling="yarn", factor=2.0), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            rope_frequencies(device="cpu", **bad)


def test_rope_at_refuses_cpu_tensors():
    from torchplusplus_amd.dlops.rope import rope_apply_at
    q = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        rope_apply_at(q, None, torch.zeros(2, dtype=torch.int32), torch.ones(32, dtype=torch.float64))


@pytest.mark.gpu
def test_rope_at_refusals(dev):
    from torchplusplus_amd.dlops.rope import rope_apply_at, rope_apply_at_
    q = torch.zeros(2, 3, 2, 64, dtype=torch.float16, device=dev)
    p, f = torch.zeros(2, 3, dtype=torch.int32, device=dev), torch.ones(32, dtype=torch.float64, device=dev)
    for bad in ((q.float(), None, p, f), (q, q.bfloat16(), p, f), (q, q[:, :2], p, f), (q, None, p[:, :2], f),
                (q, None, p.float(), f), (q, None, p, f.float()), (q, None, p, torch.cat([f, f])),
                (q, None, p, f[:0]), (q[0], None, p, f), (q.transpose(2, 3), None, p, f[:1]),
                (q, None, p.cpu(), f)):
        with pytest.raises(RuntimeError):
            rope_apply_at(*bad)
    with pytest.raises(RuntimeError, match="overlap"):
        rope_apply_at_(q[:, :1].expand(2, 3, 2, 64), None, p, f)
    with pytest.raises(RuntimeError, match="one tensor"):
        rope_apply_at_(q, q, p, f)
    assert rope_apply_at(q[:, :0], None, p[:, :0], f)[0].shape == (2, 0, 2, 64)
