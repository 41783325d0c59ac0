"""Whether the tolerance of attention over a long, split cache can fail: mistakes planted in the reference, on the CPU."""
import pytest
import torch

from test_paged_accuracy_gpu import BF16, FP16, rounded_attention64


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64), (BF16, 256)], ids=str)
def test_a_lost_tile_exceeds_the_tolerance(dtype, D):
    g = torch.Generator().manual_seed(53)
    n = 20001
    q, k, v = (torch.randn(m, D, generator=g).to(dtype).double() for m in (4, n, n))
    o, lse, tol, tl = rounded_attention64(q, k, v, D ** -0.5, dtype, -(-n // 32) + 315)
    p = torch.exp2(q @ k.T * (D ** -0.5 * 1.4426950408889634) - lse[:, None])
    # (results are rounded to `dtype`: half a step of them is in the tolerance already, another half is what hides a mistake)
    hides = tol + 2.0 ** (-8 if dtype == BF16 else -11) * o.abs()
    for at in torch.randint(0, n - 64, (50,), generator=g).tolist():
        there, next_ = slice(at, at + 32), slice(at + 32, at + 64)
        lost = p[:, there] @ v[there]
        assert (lost.abs() > hides).any(), f"values {at} .. {at + 31} lost"
        moved = p[:, there] @ (v[next_] - v[there])
        assert (moved.abs() > hides).any(), f"values {at} .. {at + 31} taken from the tile behind them"
        assert (torch.log2(1 - p[:, there].sum(1)).abs() > tl).all(), f"keys {at} .. {at + 31} not seen"
