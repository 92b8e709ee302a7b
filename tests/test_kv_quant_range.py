"""Cache codes at the ends of the input types: what is finite reads back finite."""
import pytest
import torch

from oracle import speculative as osp
from torchplusplus_amd.llmops.kvcache import kv_quant_append, kv_quant_read

CODES = [torch.float8_e4m3fn, torch.int8]


def rows(dtype, d):
    """Rows that end at and near the type's largest value, of both signs."""
    top = torch.finfo(dtype).max
    x = torch.randn(1, 12, 2, d, generator=torch.Generator().manual_seed(5)).double()
    x = x / x.abs().amax(-1, keepdim=True)
    part = torch.tensor([1.0, 0.998, 0.98, 0.97, 0.95, 0.94, 0.93, 0.9, 0.88, 0.75, 0.6, 0.5]).view(1, 12, 1, 1)
    return (x * part * top).clamp(-top, top).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_finite_rows_read_back_finite(dev, dtype, code, d):
    """The error is at most 2^-4 of the value (e4m3; below its normal codes, and in
    int8, half a step, 2^-8 and 2^-1 of the row's power of two)."""
    x = rows(dtype, d)
    assert bool(torch.isfinite(x).all()) and float(x.abs().max()) == torch.finfo(dtype).max
    codes = [torch.zeros(1, 2, 16, d, dtype=torch.uint8, device=dev).view(code) for _ in "kv"]
    exps = [torch.full((1, 2, 16), 127, dtype=torch.uint8, device=dev) for _ in "kv"]
    kv_quant_append(x.to(dev), (-x).to(dev), *codes, *exps, 0)
    want, we = osp.quantise(x, code)
    assert torch.equal(exps[0][:, :, :12].cpu(), we.transpose(1, 2))
    assert torch.equal(codes[0][:, :, :12].float().cpu(), want.transpose(1, 2).float())
    step = torch.exp2(we.double() - 127).unsqueeze(-1)
    for out, sign in zip(kv_quant_read(*codes, *exps, 12, dtype), (1, -1)):
        y = sign * out.transpose(1, 2).cpu().double()
        assert bool(torch.isfinite(y).all())
        tol = x.double().abs() * 2.0 ** -4 + step * 2.0 ** -8 if code != torch.int8 else step * 0.5
        assert bool(((y - x.double()).abs() <= tol).all())


@pytest.mark.parametrize("code", CODES)
def test_the_oracle_keeps_finite_rows_finite(code):
    x = rows(torch.bfloat16, 64)
    c, e = osp.quantise(x, code)
    v = osp.values(c, e)
    assert bool(torch.isfinite(v.bfloat16()).all())
    inf = x.clone()
    inf[0, 0, 0, 3] = float("inf")
    assert int(osp.quantise(inf, code)[1][0, 0, 0]) == 255
