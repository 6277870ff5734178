"""e4m3 caches hold value / scale, the fp32 quotient rounded once more: bit for bit what PyTorch's division and conversion
give, for scales that are no powers of two and values at the borders between two e4m3 numbers."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def _append(ext, x, kvh, hd, k_scale, v_scale):
    """x [T, 2 * kvh * hd] as keys and values behind one zero query head, neither normed nor rotated."""
    T = x.shape[0]
    pools = [torch.zeros(-(-T // 16), kvh, 16, hd, device="cuda").to(R.DT["fp8"]) for _ in range(2)]
    qkv = torch.cat([torch.zeros(T, hd, dtype=x.dtype, device="cuda"), x], 1)
    at = torch.arange(T, device="cuda")
    ext.qk_norm_rope_append(qkv, None, None, at, at, *pools, 1, eps=None, k_scale=k_scale, v_scale=v_scale)
    return [p.transpose(1, 2).flatten(0, 1)[:T] for p in pools]


def _same(got, x, scale):
    want = (x.float() / torch.tensor(scale, device="cuda")).clamp(-448, 448).to(R.DT["fp8"])
    return torch.equal(R.raw(got), R.raw(want.view(got.shape)))


@pytest.mark.parametrize("scale", [0.3, 0.07, 1.7, 0.25, 3e-5])
@pytest.mark.parametrize("T", [96, 1536])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_e4m3_is_the_quotient(ext, dtype, T, scale):
    """Every finite value of the type that the scale brings into e4m3's range, and the values next to scale * border."""
    kvh, hd = 2, 128
    every = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    every = every[torch.isfinite(every.float()) & (every.float().abs() <= 500 * scale)]
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(R.DT["fp8"]).double()
    border = torch.cat([(codes[1:] + codes[:-1]) / 2, codes]).cuda() * scale
    border = border.to(dtype)
    at = torch.cat([border.view(torch.int16) + d for d in (-1, 0, 1)]).view(dtype)
    values = torch.cat([every, at, -at])
    values = values[torch.isfinite(values.float())]
    size = T * 2 * kvh * hd
    for part in values.split(size):
        x = part.repeat(-(-size // part.numel()))[:size].view(T, -1)
        k, v = _append(ext, x, kvh, hd, scale, scale)
        assert _same(k, x[:, :kvh * hd], scale) and _same(v, x[:, kvh * hd:], scale)


def test_append_e4m3_smallest_scale(ext):
    """A scale whose reciprocal is no finite number: zeros stay zeros, the rest saturates."""
    x = torch.zeros(4, 2 * 128, dtype=torch.float16, device="cuda")
    x[1::2] = 1.0
    for got in _append(ext, x, 1, 128, 1e-39, 1e-39):
        assert (got.float()[::2] == 0).all() and (got.float()[1::2] == 448).all()
