"""What attention over pages keeps of its probabilities and values, on the GPU against 64 bits, with inputs that would show a lost bit.

Tolerances, from the arithmetic.  A logit in base 2 that is one product, times the scale, is off by 2^-24 of it for the scale's own
rounding and 2^-24 for the product's: e = 2^-23 |s|.  A probability is off by the factor 2^e and by the exponential's last unit, 2^-23;
what it is held in while it meets the values leaves 2^-23 of it (fp16: two pieces of 11 bits).  A sum of m terms is off by m 2^-24
of the sum of their magnitudes.  One rounding to the output's type at the end: u |o| (fp16 below its normal range: 2^-25).
"""
import math

import pytest
import torch

import moda_amd

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
TINY = {BF16: 0.0, FP16: 2.0 ** -25, FP32: 0.0}
PAGE = 16


def pages_of(keys, values, dev):
    """keys, values [B, n, H, *] -> cache_k, cache_v, page_table, past (the last key is the new token's)."""
    B, n, H, _ = keys.shape
    need = -(-n // PAGE)
    table = torch.randperm(B * need, generator=torch.Generator().manual_seed(3)).int().view(B, need)
    out = []
    for x in (keys, values):
        c = torch.full((B * need, PAGE, H, x.shape[3]), math.nan, dtype=x.dtype)
        padded = torch.full((B, need * PAGE, H, x.shape[3]), math.nan, dtype=x.dtype)
        padded[:, :n] = x
        c[table.flatten().long()] = padded.view(B * need, PAGE, H, x.shape[3])
        out.append(c.to(dev))
    return (*out, table.to(dev), torch.full((B,), n - 1, dtype=torch.int32, device=dev))


def within(got, want, tol, what):
    ok = bool(((got - want).abs() <= tol).all())
    assert ok, f"{what}: {float(((got - want).abs() / tol).max())} times what is allowed"


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_probabilities_keep_their_bits(dtype, gpu_device):
    """One key's weighted value against three others of the opposite sign, each the rounding of what is left: the result is what a
    probability loses on its way, and the output's own rounding is out of sight."""
    g = torch.Generator().manual_seed(31)
    B, H, D, Dv = 64, 2, 8, 64
    q = torch.zeros(B, 1, H, D, dtype=dtype)
    q[..., 0] = 1
    keys, values = torch.zeros(B, 4, H, D, dtype=dtype), torch.zeros(B, 4, H, Dv, dtype=dtype)
    keys[:, 1, :, 0] = -(0.25 + 1.75 * torch.rand(B, H, generator=g)).to(dtype)
    p = torch.exp(keys[..., :1].double())  # [B, 4, H, 1]: 1, p, 1, 1
    values[:, 1] = (1 + torch.rand(B, H, Dv, generator=g)).to(dtype)
    left = p[:, 1] * values[:, 1].double()
    for i in (0, 2, 3):
        values[:, i] = (-left).to(dtype)
        left = left + values[:, i].double()
    o = moda_amd.paged_moda(q.to(gpu_device), *pages_of(keys, values, gpu_device), scale=1.0)[:, 0].double().cpu()
    want, magnitude = (p * values.double()).sum(1) / p.sum(1), (p * values.double().abs()).sum(1) / p.sum(1)
    e = 2.0 ** -23 * keys[:, 1, :, :1].double().abs() * math.log2(math.e)
    # 4 keys in at most 3 pieces, the division, the exponential and the pieces of the sum under it
    tol = U[dtype] * want.abs() + (math.log(2) * e + 2 * 2.0 ** -23 + (12 + 2) * 2.0 ** -24) * magnitude + TINY[dtype]
    within(o, want, tol, str(dtype))
