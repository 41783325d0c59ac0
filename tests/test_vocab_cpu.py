"""Refusals of the embedding and of the cross entropy over a vocabulary: the C entries with arguments that never reach a device, and the Python
functions on tensors that are not on one."""
import ctypes
from ctypes import c_float, c_int32, c_int64, c_size_t, c_void_p

import pytest
import torch

import moda_amd
from moda_amd import _lib

EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = -1, -2, -3, -4


class Args(ctypes.Structure):
    _fields_ = [("struct_size", c_int32), ("dtype", c_int32), ("rows", c_int64), ("vocab", c_int64), ("width", c_int64),
                ("x", c_void_p), ("weight", c_void_p), ("targets", c_void_p), ("ld_x", c_int64), ("ld_weight", c_int64), ("ignore_index", c_int64),
                ("targets64", c_int32), ("reduction", c_int32), ("scale", c_float), ("reserved", c_int32),
                ("loss", c_void_p), ("lse", c_void_p), ("d_loss", c_void_p), ("dx", c_void_p), ("d_weight", c_void_p),
                ("ld_dx", c_int64), ("ld_d_weight", c_int64)]


def args(**change):
    a = Args(ctypes.sizeof(Args), 0, 100, 1000, 64, 4096, 8192, 16384, 64, 64, -100, 1, 2, 1.0, 0, 256, 512, 256, 4096, 8192, 64, 64)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.fixture(scope="module")
def lib():
    lib = _lib.load()
    for name in ("moda_hip_vocab_loss_fwd", "moda_hip_vocab_loss_bwd"):
        getattr(lib, name).argtypes = [c_void_p, c_void_p, c_size_t, c_void_p]
        getattr(lib, name + "_workspace_bytes").argtypes = [c_void_p]
        getattr(lib, name + "_workspace_bytes").restype = c_size_t
    lib.moda_hip_embed_rows.argtypes = [c_int32, c_void_p, c_int32, c_int64, c_void_p, c_int64, c_int64, c_int64, c_float, c_void_p, c_int64, c_void_p]
    lib.moda_hip_embed_grad.argtypes = [c_int32, c_void_p, c_int32, c_int64, c_void_p, c_int64, c_int64, c_int64, c_float, c_void_p, c_int64, c_void_p, c_size_t,
                                        c_void_p]
    lib.moda_hip_embed_grad_workspace_bytes.argtypes = [c_int64, c_int64, c_int64]
    lib.moda_hip_embed_grad_workspace_bytes.restype = c_size_t
    return lib


@pytest.mark.parametrize("change,rc", [
    (dict(struct_size=8), EINVAL), (dict(dtype=3), EINVAL), (dict(rows=-1), EINVAL), (dict(vocab=0), EINVAL), (dict(width=0), EINVAL),
    (dict(targets=None), EINVAL), (dict(reduction=3), EINVAL), (dict(ld_x=-1), EINVAL), (dict(scale=float("inf")), EINVAL),
    (dict(scale=float("nan")), EINVAL), (dict(x=None), EINVAL), (dict(weight=None), EINVAL), (dict(lse=None), EINVAL),
    (dict(targets=16388), EALIGN), (dict(x=4097), EALIGN), (dict(weight=8193), EALIGN), (dict(lse=514), EALIGN),
    (dict(rows=1 << 24), EUNSUPPORTED), (dict(vocab=(1 << 31) - 256), EUNSUPPORTED), (dict(width=(1 << 16) + 1), EUNSUPPORTED)])
@pytest.mark.parametrize("which", ["fwd", "bwd"])
def test_loss_arguments(lib, which, change, rc):
    a = args(**change)
    assert getattr(lib, "moda_hip_vocab_loss_" + which)(ctypes.byref(a), 256, 1 << 40, None) == rc
    if rc == EUNSUPPORTED or "struct_size" in change:
        assert getattr(lib, f"moda_hip_vocab_loss_{which}_workspace_bytes")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("which", ["fwd", "bwd"])
def test_loss_workspace(lib, which):
    a = args()
    need = getattr(lib, f"moda_hip_vocab_loss_{which}_workspace_bytes")(ctypes.byref(a))
    run = getattr(lib, "moda_hip_vocab_loss_" + which)
    assert need > 0
    assert run(ctypes.byref(a), 256, need - 1, None) == EWORKSPACE
    assert run(ctypes.byref(a), None, need, None) == EWORKSPACE
    assert run(ctypes.byref(a), 264, need, None) == EALIGN


def test_backward_arguments(lib):
    run = lambda **c: lib.moda_hip_vocab_loss_bwd(ctypes.byref(args(**c)), 256, 1 << 40, None)  # noqa: E731
    if torch.cuda.is_available():
        pytest.skip("pointers are made up")
    for change, rc in [(dict(d_loss=None), EINVAL), (dict(ld_dx=63), EINVAL), (dict(ld_d_weight=63), EINVAL), (dict(dx=4097), EALIGN), (dict(d_loss=258), EALIGN)]:
        assert run(**change) in (rc, -6)  # (-6: the device is asked for first)


@pytest.mark.parametrize("which,change,rc", [
    ("fwd", dict(loss=None), EINVAL), ("fwd", dict(loss=None, reduction=0), EINVAL), ("fwd", dict(loss=None, rows=0), EINVAL), ("fwd", dict(loss=258), EALIGN),
    ("bwd", dict(d_loss=None), EINVAL), ("bwd", dict(ld_dx=63), EINVAL), ("bwd", dict(ld_d_weight=63), EINVAL), ("bwd", dict(dx=4097), EALIGN),
    ("bwd", dict(d_weight=8193), EALIGN), ("bwd", dict(d_weight=8194, dtype=2), EALIGN), ("bwd", dict(d_loss=258), EALIGN)])
def test_arguments_of_one_pass(lib, which, change, rc):
    """Refused before anything asks for a device, so that the code is the argument's own on any machine."""
    assert getattr(lib, "moda_hip_vocab_loss_" + which)(ctypes.byref(args(**change)), 256, 1 << 40, None) == rc


def test_workspaces_stay_bounded(lib):
    """Of pieces: a GiB for the logits' gradient, as much for the weight laid out anew, whatever the vocabulary."""
    for dtype in (0, 2):
        sizes = [lib.moda_hip_vocab_loss_bwd_workspace_bytes(ctypes.byref(args(dtype=dtype, rows=1 << 15, width=1024, ld_x=1024, ld_weight=1024, ld_dx=1024,
                                                                               ld_d_weight=1024, vocab=v))) for v in (1 << 17, 1 << 20, 1 << 24)]
        assert max(sizes) < 6 << 30, sizes


@pytest.mark.parametrize("dtype", [0, 2])
@pytest.mark.parametrize("rows", [1, 4096, 1 << 15])
def test_forward_workspaces_stay_bounded(lib, dtype, rows):
    """Statistics of a piece of the vocabulary at a time (2 GiB at most, 8 bytes for each row and tile of words), and of fp32 weights a GiB laid out anew."""
    need = lambda v: lib.moda_hip_vocab_loss_fwd_workspace_bytes(ctypes.byref(args(dtype=dtype, rows=rows, width=1024, ld_x=1024, ld_weight=1024, vocab=v)))  # noqa: E731
    sizes = [need(v) for v in (1 << 17, 1 << 20, 1 << 24, 1 << 30)]
    assert max(sizes) < (2 << 30) + (1 << 30) + rows * 1024 * 6 + (1 << 20), sizes
    assert sizes[3] <= 2 * sizes[2], sizes  # pieces of 2^21 words at most


@pytest.mark.parametrize("change,rc", [
    (dict(dtype=5), EINVAL), (dict(n=-1), EINVAL), (dict(vocab=0), EINVAL), (dict(width=0), EINVAL), (dict(tokens=None), EINVAL), (dict(at=None), EINVAL),
    (dict(out=None), EINVAL), (dict(ld_out=7), EINVAL), (dict(ld=-1), EINVAL), (dict(scale=float("nan")), EINVAL), (dict(tokens=4), EALIGN),
    (dict(at=33), EALIGN), (dict(out=65), EALIGN), (dict(n=1 << 30), EUNSUPPORTED), (dict(vocab=(1 << 31) - 256), EUNSUPPORTED), (dict(width=1 << 24, ld_out=1 << 24), EUNSUPPORTED)])
def test_embedding_arguments(lib, change, rc):
    c = dict(dtype=0, tokens=8, n=10, at=32, ld=8, vocab=50, width=8, scale=1.0, out=64, ld_out=8)
    c.update(change)
    head = (c["dtype"], c["tokens"], 1, c["n"], c["at"], c["ld"], c["vocab"], c["width"], c["scale"], c["out"], c["ld_out"])
    assert lib.moda_hip_embed_rows(*head, None) == rc
    assert lib.moda_hip_embed_grad(*head, 256, 1 << 40, None) == rc


def test_embedding_workspace(lib):
    need = lib.moda_hip_embed_grad_workspace_bytes(10, 50, 8)
    assert need > 0
    for ws, size, rc in ((None, need, EWORKSPACE), (256, need - 1, EWORKSPACE), (257, need, EALIGN)):
        assert lib.moda_hip_embed_grad(0, 8, 1, 10, 32, 8, 50, 8, 1.0, 64, 8, ws, size, None) == rc
    assert lib.moda_hip_embed_grad_workspace_bytes(1 << 30, 50, 8) == 0


def test_no_cpu_path():
    w, t = torch.zeros(5, 8), torch.zeros(3, dtype=torch.long)
    for call in (lambda: moda_amd.embed_tokens(t, w), lambda: moda_amd.embed_tokens_bwd(t, torch.zeros(3, 8), 5), lambda: moda_amd.linear_cross_entropy(torch.zeros(3, 8), w, t),
                 lambda: moda_amd.linear_cross_entropy_fwd(torch.zeros(3, 8), w, t),
                 lambda: moda_amd.linear_cross_entropy_bwd(torch.zeros(3, 8), w, t, torch.zeros(3), torch.zeros(()))):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


def test_stack_with_a_vocabulary():
    plain, tied, apart = (moda_amd.MoDAStack(32, 1, 4, 2, **k) for k in ({}, {"vocab": 50}, {"vocab": 50, "tied": False}))
    more = lambda m: sorted(set(m.state_dict()) - set(plain.state_dict()))  # noqa: E731
    assert more(tied) == ["embedding", "out_norm.bias", "out_norm.weight"] and more(apart) == ["embedding", "head", "out_norm.bias", "out_norm.weight"]
    with pytest.raises(ValueError, match="at least one word"):
        moda_amd.MoDAStack(32, 1, 4, 2, vocab=0)
    with pytest.raises(AssertionError, match="construct with vocab"):
        plain(torch.zeros(1, 3, dtype=torch.long))
    with pytest.raises(AssertionError, match="construct with vocab"):
        plain.nll(torch.zeros(1, 3, 32), torch.zeros(1, 3, dtype=torch.long))
