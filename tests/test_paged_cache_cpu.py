"""What a cache of pages counts and refuses, without a GPU."""
import ctypes

import pytest
import torch

import moda_amd
from moda_amd import _lib

from test_paged_cpu import AT, EINVAL, AppendC, pages, strides


def cache(**kw):
    args = dict(layers=1, n_pages=6, page_size=16, H=1, D=8, dtype=torch.float32, device="cpu", batch=3, max_tokens=64)
    return moda_amd.PagedKVCache(**{**args, **kw})


def test_prompts_need_empty_sequences_and_pages():
    c = cache()
    for b, n in enumerate((33, 16, 0)):
        c.reserve(b, n)
    lens = lambda *n: torch.tensor(n, dtype=torch.int32)  # noqa: E731
    c.check_prompts(33, lens(33, 16, 0))
    c.check_prompts(40, lens(40, 9, -5))  # three pages; counts below zero are none
    c.check_prompts(0)
    for n, l in ((33, None), (33, lens(33, 17, 0)), (49, lens(49, 0, 0)), (33, lens(1, 1, 1)), (65, lens(99, 0, 0))):
        with pytest.raises(RuntimeError, match="pages"):
            c.check_prompts(n, l)
    c.past.copy_(lens(0, 1, -3))
    c.check_prompts(33, lens(33, 0, 0))
    with pytest.raises(RuntimeError, match="empty"):
        c.check_prompts(33, lens(33, 1, 0))
    c.release(1)
    c.reserve(1, 16)
    c.check_prompts(33, lens(33, 1, 0))
    with pytest.raises(AssertionError):
        c.check_prompts(33, lens(33, 1))


def test_pages_that_come_late_hold_no_tokens():
    """Positions that were counted without a page were dropped: the page that would hold them now has not been written."""
    c = cache()
    c.reserve(0, 20), c.reserve(1, 16), c.reserve(2, 1)
    c.past.copy_(torch.tensor([35, 9, 17], dtype=torch.int32))
    c.reserve(0, 32)  # has them already
    assert c.past.tolist() == [35, 9, 17]
    c.reserve(0, 40)
    c.reserve(1, 17)
    assert c.past.tolist() == [32, 9, 17]
    c.release(1)
    c.reserve(2, 30)
    assert c.past.tolist() == [32, 0, 16]


def test_arrays_of_no_sequences_may_be_null():
    lib, s = _lib.load(), strides(128, 128, 64)
    a = AppendC(struct_size=ctypes.sizeof(AppendC), k=AT, v=AT, sk=s, sv=s)
    for kw, code in ((dict(B=0, table=None, past=None), 0), (dict(B=0, table=None, past=None, cu_seqlens=AT, total_tokens=0), 0),
                     (dict(table=None), EINVAL), (dict(past=None), EINVAL), (dict(B=0, k_pages=None), EINVAL)):
        assert lib.moda_hip_paged_append(ctypes.byref(pages(**kw)), ctypes.byref(a), None, None) == code, kw
