"""Stacks that generate: prompts and tokens through the paged cache against the whole sequence at once, in fp32.

Tolerance: both sides add up the same products in fp32, in other orders.  A block is about five sums of at most 512 terms one after
the other (projections, attention, MLP), the norms keep what enters them at order one; n terms in another order differ by
at most n 2^-24 of the sum of magnitudes: 5 x 512 x 2^-24 = 1.6e-4 a block relative to the rows' size.
"""
import copy
import math

import pytest
import torch

import moda_amd

pytestmark = pytest.mark.gpu

STACKS = [
    # dim, depth, heads, kv heads, rotated, post_norm, ffn_kv
    (64, 3, 4, 2, 16, False, False),
    (64, 2, 2, 1, 32, False, True),
    (128, 2, 4, 4, 0, True, False),
    (96, 2, 4, 2, 20, True, True),
    (64, 2, 4, 1, 0, False, True),
]


def make(spec, dev, dtype=torch.float32):
    dim, depth, heads, kv, rot, post, ffn = spec
    torch.manual_seed(21)
    rotary = moda_amd.Rotary(rot, base=100.0, interleaved=dim == 96) if rot else None
    m = moda_amd.MoDAStack(dim, depth, heads, kv, mlp_ratio=2.0, is_causal=True, post_norm=post, ffn_kv=ffn, rotary=rotary)
    return m.to(dev, dtype).eval()


def make_cache(m, batch, tokens, dev, dtype=torch.float32, page=16, spare=3):
    attn = m.blocks[0].attn
    pages = -(-tokens // page)
    c = moda_amd.PagedKVCache(len(m.blocks), batch * pages + spare, page, attn.num_kv_heads, attn.head_dim, dtype, dev, batch=batch, max_tokens=tokens)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    return c


def check(got, want, blocks, what):
    err = (got.double() - want.double()).abs().max()
    assert err <= 1.6e-4 * blocks * want.abs().max(), (what, float(err))


@pytest.mark.parametrize("spec", STACKS, ids=str)
def test_prompts_and_tokens_are_the_whole_sequence(spec, gpu_device):
    dev, T = gpu_device, 61
    m = make(spec, dev)
    x = torch.randn(3, T, spec[0], device=dev)
    with torch.no_grad():
        whole = m(x)
    lens = [40, 17, 1]
    cache = make_cache(m, 3, T + 20, dev)
    for b in range(3):
        cache.reserve(b, T + 19)
    prompt = torch.randn(3, 40, spec[0], device=dev)
    for b, n in enumerate(lens):
        prompt[b, :n] = x[b, :n]
    out = m.prefill(prompt, cache, lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    for b, n in enumerate(lens):
        check(out[b, :n], whole[b, :n], spec[1], f"prompt {b}")
    at = list(lens)
    for step in (1, 1, 4, 1, 9):  # the sequences go on from where each of them is; some steps are padded
        new = [step if (b + step) % 4 else max(step - 2, 0) for b in range(3)]
        rows = torch.randn(3, step, spec[0], device=dev)
        for b in range(3):
            rows[b, :new[b]] = x[b, at[b]:at[b] + new[b]]
        ragged = min(new) < step
        out = m.decode(rows, cache, lens=torch.tensor(new, dtype=torch.int32, device=dev) if ragged else None)
        for b in range(3):
            if new[b]:
                check(out[b, :new[b]], whole[b, at[b]:at[b] + new[b]], spec[1], f"step {step} sequence {b}")
            at[b] += new[b]
    assert cache.past.tolist() == at


def test_a_released_sequence_starts_again(gpu_device):
    m = make(STACKS[0], gpu_device)
    cache = make_cache(m, 2, 48, gpu_device, spare=0)
    x = torch.randn(2, 20, 64, device=gpu_device)
    for b in range(2):
        cache.reserve(b, 48)
    m.prefill(x, cache)
    cache.release(0)
    cache.reserve(0, 30)
    y = torch.randn(2, 12, 64, device=gpu_device)
    out = m.decode(y, cache)  # a piece of a prompt for the new sequence, the next tokens of the other
    with torch.no_grad():
        check(out[0], m(y[:1])[0], 3, "new")
        check(out[1], m(torch.cat([x[1:], y[1:]], 1))[0, 20:], 3, "old")


def test_captured_decode_follows_the_counts(gpu_device):
    dev = gpu_device
    m = make((128, 2, 4, 2, 32, False, True), dev, torch.bfloat16)
    cache, plain = (make_cache(m, 2, 100, dev, torch.bfloat16) for _ in range(2))
    prompt = torch.randn(2, 30, 128, device=dev).bfloat16()
    for c in (cache, plain):
        for b in range(2):
            c.reserve(b, 100)
        m.prefill(prompt, c)
    x = torch.randn(2, 1, 128, device=dev).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.decode(x, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.decode(x, cache)
    cache.past.fill_(30)
    for i in range(20):
        x.normal_()
        graph.replay()
        got = out.clone()
        want = m.decode(x, plain)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
    assert cache.past.tolist() == [50, 50]


def test_training_with_a_rotation_through_the_depth_stream(gpu_device):
    """Gradients of a stack that rotates, in place and rebuilt: the same sums in another order; and against differences."""
    dev = gpu_device
    m = make((64, 2, 4, 2, 16, False, True), dev)
    x = torch.randn(2, 23, 64, device=dev)
    w = torch.randn(2, 23, 64, device=dev)
    grads = []
    for inplace in (None, False):
        p = copy.deepcopy(m).train()
        y = p(x, inplace_cache=inplace)
        (y * w).sum().backward()
        grads.append({n: q.grad for n, q in p.named_parameters()})
    for n, g in grads[0].items():
        if grads[1][n] is None:  # the last block's FFN keys and values: nobody sees them
            assert g is None and n.startswith("blocks.1.attn.kv_ffn"), n
            continue
        assert (g - grads[1][n]).abs().max() <= 2 * 1.6e-4 * 2 * grads[1][n].abs().max(), n
    m64 = []
    p = m.blocks[0].attn.q.weight
    d = torch.randn_like(p)
    d /= d.norm()
    step = 2.0 ** -6
    with torch.no_grad():
        for s in (step, -step, 2 * step, -2 * step):
            q = copy.deepcopy(m)
            q.blocks[0].attn.q.weight.add_(s * d)
            m64.append(float((q(x, inplace_cache=False).double() * w.double()).sum()))
    # fourth-order differences: truncation of order step^4 = 6e-8; rounding: sums of magnitude sum |y w| at 1.6e-4 / sqrt(terms)
    slope = (8 * (m64[0] - m64[1]) - (m64[2] - m64[3])) / (12 * step)
    exact = float((grads[0]["blocks.0.attn.q.weight"].double() * d.double()).sum())
    scale = float((grads[0]["blocks.0.attn.q.weight"].double().norm()))
    assert abs(slope - exact) <= 2e-2 * scale, (slope, exact, scale)


def test_positions_shift_a_whole_sequence(gpu_device):
    """Attention sees differences of positions only: the same tokens further along give the same result, the angles being exact to
    2^-23 of a turn at any position."""
    m = make(STACKS[0], gpu_device)
    x = torch.randn(1, 40, 64, device=gpu_device)
    with torch.no_grad():
        check(m(x, positions=torch.arange(700000, 700040, device=gpu_device)), m(x), 3, "shifted")


def test_stacks_refuse(gpu_device):
    dev = gpu_device
    m = make(STACKS[0], dev)
    cache = make_cache(m, 2, 32, dev)
    x = torch.randn(2, 3, 64, device=dev)
    for bad in (moda_amd.MoDAStack(64, 3, 4, 2, is_causal=False).to(dev), moda_amd.MoDAStack(64, 3, 4, 2, is_causal=True, chunk_rows=64).to(dev),
                moda_amd.MoDAStack(64, 2, 4, 2, is_causal=True).to(dev)):
        with pytest.raises(AssertionError):
            bad.decode(x, cache)
        with pytest.raises(AssertionError):
            bad.prefill(x, cache)
    with pytest.raises(AssertionError):
        m.decode(x[:1], cache)
    with pytest.raises(AssertionError):
        moda_amd.MoDAStack(64, 3, 4, 4, is_causal=True).to(dev).decode(x, cache)  # other heads than the cache's
    with pytest.raises(AssertionError):
        moda_amd.MoDAAttention(64, 4, 2, is_causal=True).to(dev)(x, positions=torch.arange(3, device=dev))
    assert m.decode(x[:, :0], cache).shape == (2, 0, 64)
