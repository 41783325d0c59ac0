"""Calls of the rotation and the paged cache that the documentation allows or refuses at their edges, on the GPU."""
import math

import pytest
import torch

import moda_amd

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def pages(dev, n=4, page=16, H=2, D=64, B=1, width=3, dtype=BF16):
    """cache_k, cache_v, page_table, past of empty sequences whose first pages are 0, 1, .."""
    ck, cv = (torch.zeros(n, page, H, D, dtype=dtype, device=dev) for _ in range(2))
    return ck, cv, torch.arange(B * width, dtype=torch.int32, device=dev).view(B, width), torch.zeros(B, dtype=torch.int32, device=dev)


def test_forward_mode_derivatives_are_refused(gpu_device):
    """A tangent that a call cannot pass on is an error, not lost; without one the same calls run."""
    dev = gpu_device
    z = lambda *s: torch.zeros(*s, dtype=BF16, device=dev)  # noqa: E731
    ck, cv, table, past = pages(dev)
    q, k = z(1, 4, 2, 64), z(1, 1, 2, 64)

    def attend(q=q, ck=ck, cv=cv, kd=None, vd=None):
        return moda_amd.paged_moda(q, ck, cv, table, past, moda_group_num=4, cached_k=kd, cached_v=vd)

    def append(k=k, v=k, ck=ck, cv=cv, q=None):
        return moda_amd.paged_append(k, v, ck, cv, table, past, q=q, rotary=moda_amd.Rotary(64))

    def plain(q=k):
        return moda_amd.paged_attn(q, ck, cv, table, past)

    attend(), append(), plain(), append(q=k)
    fw = torch.autograd.forward_ad
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fw.dual_level():
            dual = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
            for f, name in ((attend, "q"), (attend, "ck"), (attend, "cv"), (append, "k"), (append, "v"), (append, "ck"), (append, "q"), (plain, "q")):
                x = {"q": q if f is attend else k, "ck": ck, "cv": cv, "k": k, "v": k}[name]
                with pytest.raises(AssertionError, match="forward-mode"):
                    f(**{name: dual(x)})
            with pytest.raises(AssertionError, match="forward-mode"):
                attend(kd=dual(k), vd=k)
            attend(), append(), plain()
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        moda_amd.apply_rotary(fw.make_dual(k, torch.ones_like(k)), None, moda_amd.Rotary(64))
