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


def stack(dev, depth=2, rotary=True):
    torch.manual_seed(41)
    return moda_amd.MoDAStack(64, depth, 4, 2, mlp_ratio=2.0, is_causal=True, rotary=moda_amd.Rotary(16) if rotary else None).to(dev).eval()


def stack_cache(dev, batch=2, n_pages=8, max_tokens=64):
    return moda_amd.PagedKVCache(2, n_pages, 16, 2, 16, torch.float32, dev, batch=batch, max_tokens=max_tokens)


def test_prefill_refuses_sequences_that_have_tokens_or_no_pages(gpu_device):
    """Keys rotated from position zero would lie behind those that are there; tokens without pages would be gone."""
    dev = gpu_device
    m, c = stack(dev), stack_cache(dev)
    x = torch.randn(2, 20, 64, device=dev)
    with pytest.raises(RuntimeError, match="pages"):
        m.prefill(x, c)
    c.reserve(0, 20)
    with pytest.raises(RuntimeError, match="pages"):
        m.prefill(x, c)
    first = torch.tensor([20, 0], dtype=torch.int32, device=dev)
    m.prefill(x, c, lens=first)
    assert c.past.tolist() == [20, 0]
    c.reserve(0, 64), c.reserve(1, 20)
    with pytest.raises(RuntimeError, match="empty"):
        m.prefill(x, c)
    m.prefill(x, c, lens=20 - first)  # the other one, beside a sequence that goes on
    assert c.past.tolist() == [20, 20]
    c.release(0)
    c.reserve(0, 20)
    m.prefill(x, c, lens=first)
    with pytest.raises(AssertionError):
        m.prefill(x, c, lens=first[:1])


def test_counts_of_new_tokens_are_bounded_everywhere(gpu_device):
    """More real tokens than the call has, or fewer than none, count as all and none: in what is stored, seen and counted, also captured."""
    dev = gpu_device
    m = stack(dev)
    x, y = torch.randn(2, 20, 64, device=dev), torch.randn(2, 3, 64, device=dev)
    out = []
    for lens in ([50, 20], [20, 20]):
        c = stack_cache(dev)
        c.k.fill_(math.nan), c.v.fill_(math.nan)
        for b in range(2):
            c.reserve(b, 64)
        r = [m.prefill(x, c, lens=torch.tensor(lens, dtype=torch.int32, device=dev))]
        r.append(m.decode(y, c, lens=torch.tensor([9, -4], dtype=torch.int32, device=dev))[:1])
        assert c.past.tolist() == [23, 20]
        r.append(m.decode(y, c))
        out.append(r)
    for a, b in zip(*out):
        assert torch.equal(a, b) and a.isfinite().all()


def test_captured_prefill(gpu_device):
    """Nothing waits for the device while a graph is captured; counts of new tokens are bounded there too."""
    dev = gpu_device
    m, c = stack(dev), stack_cache(dev)
    for b in range(2):
        c.reserve(b, 40)
    x, lens = torch.randn(2, 20, 64, device=dev), torch.tensor([20, 7], dtype=torch.int32, device=dev)
    m.prefill(x, c, lens=lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.prefill(x, c, lens=lens)
    for n in ([33, 5], [1, 0], [-2, 20]):
        x.normal_()
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        c.past.zero_()
        graph.replay()
        kept = got.clone()
        assert c.past.tolist() == [min(max(i, 0), 20) for i in n]
        c.past.zero_()
        want = m.prefill(x, c, lens=lens)
        assert torch.equal(kept, want)


def test_tokens_without_a_page_are_never_read(gpu_device):
    """A sequence that ran past its pages goes on behind what is stored once it has more: nothing of the pages' former contents is seen."""
    dev = gpu_device
    m, c = stack(dev, rotary=False), stack_cache(dev, batch=1)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    x = torch.randn(1, 24, 64, device=dev)
    c.reserve(0, 16)
    m.prefill(x[:, :14], c)
    for i in range(14, 20):  # the last four have no page
        assert m.decode(x[:, i:i + 1], c).isfinite().all()
    c.reserve(0, 40)
    assert c.past.tolist() == [16]
    out = m.decode(x[:, 20:], c)
    with torch.no_grad():
        want = m(torch.cat([x[:, :16], x[:, 20:]], 1))[:, 16:]
    # fp32 on both sides, sums of at most 128 terms in other orders through two blocks of five
    assert (out - want).abs().max() <= 2 * 5 * 128 * 2.0 ** -24 * want.abs().max()


@pytest.mark.parametrize("call", ["rotate", "append"])
def test_a_rotary_dropped_while_another_stream_uses_it(call, gpu_device):
    """The rates' memory belongs to the stream that made them: it stays theirs until the calls of other streams are done."""
    dev = gpu_device
    rot = moda_amd.Rotary(64)
    x = torch.randn(1, 3, 2, 64, device=dev).to(BF16)
    ck, cv, table, past = pages(dev)

    def run(rot):
        if call == "rotate":
            return moda_amd.apply_rotary(x, None, rot)[0]
        return moda_amd.paged_append(x, x, ck, cv, table, past, q=x, rotary=rot)

    want = run(rot)
    busy = torch.randn(8192, 8192, device=dev).to(BF16)
    out = torch.empty_like(busy)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(30):
            torch.mm(busy, busy, out=out)
        got = run(rot)
    at = rot.rates(x.device).data_ptr()
    del rot
    taken = [torch.full((32,), math.nan, dtype=torch.float64, device=dev) for _ in range(200)]
    assert not side.query(), "the other stream was done too early for this test to say anything"
    assert all(t.data_ptr() != at for t in taken)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_attention_of_2_to_the_26_rows(gpu_device):
    """As many rows as an axis of one launch has no threads for: each sequence sees its first key."""
    dev = gpu_device
    B, H, G, D = 1 << 14, 256, 16, 8
    ck, cv, _, _ = pages(dev, n=1, H=H, D=D)
    torch.manual_seed(42)
    ck[0, 0], cv[0, 0] = torch.randn(H, D, device=dev), torch.randn(H, D, device=dev)
    table, past = torch.zeros(1, 1, dtype=torch.int32, device=dev).expand(B, 1), torch.zeros(B, dtype=torch.int32, device=dev)
    q = torch.zeros(B, 1, H * G, D, dtype=BF16, device=dev)
    q[..., 0] = 1
    o, lse = moda_amd.paged_attn_fwd(q, ck, cv, table, past, scale=1.0)
    assert torch.equal(o.view(B, H, G, D), cv[0, 0][:, None].expand(B, H, G, D))
    want = ck[0, 0, :, 0].float()[:, None] * math.log2(math.e)
    assert ((lse.view(B, H, G) - want).abs() <= 2.0 ** -22 * want.abs()).all()


def test_rotation_of_2_to_the_30_tokens(gpu_device):
    """As many threads as an axis of one launch does not have."""
    T, rot = 1 << 30, moda_amd.Rotary(8)
    x = torch.randn(1, 1, 1, 8, device=gpu_device).to(BF16)
    y = moda_amd.apply_rotary(None, x.expand(1, T, 1, 8), rot)[1]
    at = torch.tensor([0, 1, 12345, (1 << 28) - 1, 1 << 28, (1 << 29) + 7, T - 2, T - 1], device=gpu_device)
    want = moda_amd.apply_rotary(None, x.expand(1, 8, 1, 8), rot, positions=at)[1]
    assert torch.equal(y[0, at], want[0])
    assert bool((y.view(torch.int16)[:, ::4096] != 0).any(-1).all())


def test_packed_tokens_of_no_sequence(gpu_device):
    """Offsets of no sequences: all rows are behind the last one, stored nowhere and returned as they are."""
    dev = gpu_device
    ck, cv, _, _ = pages(dev)
    table, past = (torch.empty(*s, dtype=torch.int32, device=dev) for s in ((0, 3), (0,)))
    x, q, kd = torch.randn(1, 5, 2, 64, device=dev).to(BF16), torch.randn(1, 10, 2, 64, device=dev).to(BF16), torch.zeros(1, 15, 2, 64, dtype=BF16, device=dev)
    q1 = moda_amd.paged_append(x, x, ck, cv, table, past, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=dev), q=q, rotary=moda_amd.Rotary(64),
                               moda_group_num=2, cached_k=kd, cached_v=kd.clone(), depth_slot=1)
    assert torch.equal(q1, q) and not ck.any() and not cv.any() and not kd.any()


def test_caches_without_a_head_dim_are_refused(gpu_device):
    """Values of no elements: the row sums would be left as their memory was."""
    dev = gpu_device
    ck, cv, table, past = pages(dev)
    q = torch.zeros(1, 1, 2, 64, dtype=BF16, device=dev)
    for k, v, x in ((ck, cv[..., :0], q), (ck[..., :0], cv, q[..., :0]), (ck[..., :0], cv[..., :0], q[..., :0])):
        with pytest.raises(AssertionError, match="head dims"):
            moda_amd.paged_moda_fwd(x, k, v, table, past)
        with pytest.raises(AssertionError, match="head dims"):
            moda_amd.paged_append(x, q[..., :v.shape[3]], k, v, table, past)


def test_tokens_without_a_page_have_their_depth_slot(gpu_device):
    """The attention of such a token still reads its own depth slots: they are written, of padded tokens they are not."""
    dev = gpu_device
    ck, cv, _, _ = pages(dev)
    table = torch.tensor([[0, -1], [9, 2]], dtype=torch.int32, device=dev)  # two pages of 16; each sequence has a hole
    past, new = torch.tensor([14, 14], dtype=torch.int32, device=dev), torch.tensor([20, 6], dtype=torch.int32, device=dev)
    k, v = (torch.randn(2, 20, 2, 64, device=dev).to(BF16) for _ in range(2))
    kd, vd = (torch.zeros(2, 20, 3, 2, 64, dtype=BF16, device=dev) for _ in range(2))
    moda_amd.paged_append(k, v, ck, cv, table, past, new_lens=new, cached_k=kd.view(2, 60, 2, 64), cached_v=vd.view(2, 60, 2, 64), depth_slot=1)
    for x, c, d in ((k, ck, kd), (v, cv, vd)):
        pages_, slots = torch.zeros_like(c), torch.zeros_like(d)
        pages_[0, 14:], pages_[2, :4] = x[0, :2], x[1, 2:6]
        slots[0, :, 1], slots[1, :6, 1] = x[0], x[1, :6]
        assert torch.equal(c, pages_) and torch.equal(d, slots)


@pytest.mark.parametrize("D", [64, 20])
@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32], ids=str)
def test_rows_of_no_sequence_stay_as_they_are(dtype, D, gpu_device):
    """To the bit: infinities, NaN and signs of zero, too."""
    dev = gpu_device
    ck, cv, table, past = pages(dev, D=64, dtype=dtype)
    R = 64 if D == 64 else 20
    q = torch.randn(1, 7, 2, 64, device=dev).to(dtype)
    q[:, 3:, 0, ::3], q[:, 3:, 1, 1::5], q[:, 3:, 1, 2::7], q[:, 0] = math.inf, -0.0, math.nan, -0.0
    cu = torch.tensor([1, 3], dtype=torch.int32, device=dev)
    for inter in (False, True):
        q1 = moda_amd.paged_append(q, q, ck, cv, table, past, cu_seqlens=cu, q=q, rotary=moda_amd.Rotary(R, interleaved=inter))
        bits = torch.int32 if dtype == torch.float32 else torch.int16
        for rows in (slice(0, 1), slice(3, 7)):
            assert torch.equal(q1[:, rows].view(bits), q[:, rows].view(bits))
        assert not torch.equal(q1[:, 2], q[:, 2])
