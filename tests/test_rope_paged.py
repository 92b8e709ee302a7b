"""qkv_rope_paged against the 64-bit form in oracle/serving.py.

Tolerance of an element made of terms of size t: its rounding eps / 2 |o| (half the
least fp16 step, 2^-25) and fp32 arithmetic, (D / 2 + 12) 2^-24 t: the norm's sum of D
squares enters by its root, then the root's reciprocal (2 units), its product with x
and w, and the rotation's two products and sum."""
import pytest
import torch

from oracle import serving as oracle


def tables(ctx, d, dtype, dev):
    a = torch.arange(ctx, dtype=torch.float64).unsqueeze(1) * 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.cat([a, a], 1)
    return torch.cos(a).to(dtype).to(dev), torch.sin(a).to(dtype).to(dev)


def make(n, hq, hk, d, page, dtype, seed, dev, norm=True, ctx=300):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(dtype).to(dev)
    pos = torch.randint(0, ctx, (n,), generator=g, dtype=torch.int32).to(dev)
    pages = n // page + 3
    slots = torch.randperm(pages * page, generator=g)[:n].to(dev)
    kp, vp = (torch.randn(pages, hk, page, d, generator=g).to(dtype).to(dev) for _ in "kv")
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(dtype).to(dev) if norm else None for _ in "qk"]
    return qkv, pos, slots, kp, vp, w


def check(q, k, kp, vp, before, qkv, pos, slots, cos, sin, hq, hk, w):
    eq, ek, ev, tq, tk = oracle.qkv_rope(qkv, pos, cos, sin, hq, hk, *w)
    dtype, d, page = qkv.dtype, cos.shape[1], kp.shape[2]
    half = torch.finfo(dtype).eps / 2
    for got, want, terms in ((q, eq, tq), (k, ek, tk)):
        tol = half * want.abs() * (1 + 2 * half) + 2.0 ** -25 + (d / 2 + 12) * 2.0 ** -24 * terms
        assert ((got.double().cpu() - want).abs() <= tol).all()
    rows = [x.cpu().clone() for x in before]
    for t in range(len(pos)):
        s = int(slots[t])
        if 0 <= s < kp.shape[0] * page and 0 <= int(pos[t]) < len(cos):
            rows[0][s // page, :, s % page], rows[1][s // page, :, s % page] = k[t].cpu(), ev[t].to(dtype)
    assert torch.equal(kp.cpu(), rows[0]) and torch.equal(vp.cpu(), rows[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hk,d,page", [(1, 16, 8, 128, 16), (33, 4, 2, 64, 32), (7, 3, 1, 256, 1024), (300, 16, 8, 128, 64),
                                            (1000, 8, 8, 64, 16)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("cs", [torch.float16, torch.float32])
def test_rows(dev, n, hq, hk, d, page, dtype, norm, cs):
    from torchplusplus_amd.llmops.paged import qkv_rope_paged
    qkv, pos, slots, kp, vp, w = make(n, hq, hk, d, page, dtype, n, dev, norm)
    cos, sin = tables(300, d, cs, dev)
    before, raw = (kp.clone(), vp.clone()), qkv.clone()
    q, k = qkv_rope_paged(qkv, pos, slots, kp, vp, cos, sin, *w)
    assert torch.equal(qkv, raw)
    check(q, k, kp, vp, before, qkv, pos, slots, cos, sin, hq, hk, w)
    q2, none = qkv_rope_paged(qkv, pos, slots, kp, vp, cos, sin, *w, with_k=False)
    assert none is None and torch.equal(q2, q)


@pytest.mark.gpu
def test_padding_and_slots_outside(dev):
    from torchplusplus_amd.llmops.paged import qkv_rope_paged
    hq, hk, d, page = 4, 2, 64, 16
    qkv, pos, slots, kp, vp, w = make(12, hq, hk, d, page, torch.bfloat16, 5, dev)
    cos, sin = tables(300, d, torch.float16, dev)
    pos[1], pos[2], pos[3] = -1, 300, 2 ** 31 - 1
    slots[4], slots[5], slots[6] = -1, kp.shape[0] * page, -2 ** 63
    qkv[2] = float("nan")
    before = (kp.clone(), vp.clone())
    q, k = qkv_rope_paged(qkv, pos, slots, kp, vp, cos, sin, *w)
    assert (q[1:4] == 0).all() and (k[1:4] == 0).all()
    qkv[2] = 1.0
    check(q, k, kp, vp, before, qkv, pos, slots, cos, sin, hq, hk, w)


@pytest.mark.gpu
def test_strides(dev):
    """A slice of a wider projection; pages that hold keys and values in turn."""
    from torchplusplus_amd.llmops.paged import qkv_rope_paged
    hq, hk, d, page = 4, 2, 128, 32
    qkv, pos, slots, kp, vp, w = make(50, hq, hk, d, page, torch.float16, 6, dev)
    cos, sin = tables(300, d, torch.float32, dev)
    wide = torch.zeros(50, qkv.shape[1] + 64, dtype=qkv.dtype, device=dev)
    wide[:, 32:-32] = qkv
    pool = torch.stack([kp, vp], 2)  # [P, H, 2, rows, D]
    before = (kp.clone(), vp.clone())
    q, k = qkv_rope_paged(wide[:, 32:-32], pos, slots, pool[:, :, 0], pool[:, :, 1], cos, sin, *w)
    check(q, k, pool[:, :, 0], pool[:, :, 1], before, qkv, pos, slots, cos, sin, hq, hk, w)


@pytest.mark.gpu
def test_refusals(dev):
    from torchplusplus_amd.llmops.paged import qkv_rope_paged
    qkv, pos, slots, kp, vp, w = make(5, 4, 2, 64, 16, torch.float16, 7, dev)
    cos, sin = tables(300, 64, torch.float16, dev)
    raw = (kp.clone(), vp.clone())
    ok = dict(qkv=qkv, positions=pos, slots=slots, k_pages=kp, v_pages=vp, cos=cos, sin=sin, q_norm=w[0], k_norm=w[1])
    odd = torch.zeros(5, qkv.shape[1] + 4, dtype=qkv.dtype, device=dev)[:, 2:-2]
    for change in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :-64]), dict(qkv=qkv[None]), dict(positions=pos.long()),
                   dict(positions=pos[:4]), dict(slots=slots.int()), dict(slots=slots[:4]), dict(slots=slots.cpu()),
                   dict(k_pages=kp.bfloat16()), dict(v_pages=vp[1:]), dict(v_pages=kp), dict(cos=cos[:, :32], sin=sin[:, :32]),
                   dict(sin=sin.float()), dict(q_norm=w[0][:32]), dict(q_norm=w[0].float()), dict(qkv=odd),
                   dict(k_pages=kp[:, :, :8], v_pages=vp[:, :, :8]), dict(cos=cos[:0], sin=sin[:0]),
                   dict(k_pages=kp[:1].expand(3, 2, 16, 64), v_pages=vp[:3])):
        with pytest.raises(RuntimeError):
            qkv_rope_paged(**{**ok, **change})
    assert torch.equal(kp, raw[0]) and torch.equal(vp, raw[1])
    q, k = qkv_rope_paged(**{**ok, "qkv": qkv[:0], "positions": pos[:0], "slots": slots[:0]})
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
