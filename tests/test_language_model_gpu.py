"""A stack with a vocabulary: both ends of a language model together with the blocks between them, training and answering, on one MI355X.

The ends' own numbers are held to their definitions in test_vocab_gpu.py; here every result is compared bit for bit with the same calls made
one by one (all kernels add in a fixed order), and the loss and its gradient once more with the definition, on the rows that the blocks make."""
import pytest
import torch

import moda_amd
from test_vocab_gpu import loss_reference, names, within, words

pytestmark = pytest.mark.gpu


def model(dtype, tied, vocab=517, dim=64, depth=2, scale=8.0, rotary=True):
    torch.manual_seed(3)
    m = moda_amd.MoDAStack(dim, depth, 4, 2, is_causal=True, rotary=moda_amd.Rotary(dim // 4) if rotary else None, vocab=vocab, tied=tied, embed_scale=scale)
    return m.to("cuda", dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=names)
@pytest.mark.parametrize("tied", [True, False])
def test_training_step(dtype, tied):
    m = model(dtype, tied)
    tokens, targets = words(150, 517, 1, 0.1).view(2, 75), words(150, 517, 2, 0.3).view(2, 75)
    loss = m.loss(tokens, targets)
    names_, params = zip(*m.named_parameters())
    grads = dict(zip(names_, torch.autograd.grad(loss, params)))
    assert loss.dtype == torch.float32 and all(g.isfinite().all() for g in grads.values())

    # the same, call by call
    x = moda_amd.embed_tokens(tokens, m.embedding.detach(), 8.0).requires_grad_()
    y = m.out_norm(m(x))
    head = (m.embedding if tied else m.head).detach()
    want, lse = moda_amd.linear_cross_entropy_fwd(y, head, targets)
    dy, dw = moda_amd.linear_cross_entropy_bwd(y, head, targets, lse, torch.ones((), device="cuda"))
    rest = [n for n in names_ if n not in ("embedding", "head")]
    dx, *others = torch.autograd.grad(y, [x] + [dict(m.named_parameters())[n] for n in rest], dy)
    de = moda_amd.embed_tokens_bwd(tokens, dx, 517, 8.0)
    assert torch.equal(loss.detach(), want)
    assert torch.equal(grads["embedding"], de + dw if tied else de) and (tied or torch.equal(grads["head"], dw))
    assert all(torch.equal(grads[n], g) for n, g in zip(rest, others))

    # and the definition, at these rows
    one = torch.ones((), device="cuda")
    ref = loss_reference(y, head, targets, 1.0, -100, "mean", one)
    for name, got in (("loss", loss.detach()), ("dx", dy), ("dw", dw)):
        within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=names)
@pytest.mark.parametrize("compute", [torch.bfloat16, torch.float16], ids=names)
def test_training_step_under_autocast(dtype, compute):
    """Parameters of any type: the norm before the loss comes out in fp32, the loss is computed in the weight's type."""
    m = model(dtype, True)
    tokens, targets = words(150, 517, 1, 0.1).view(2, 75), words(150, 517, 2, 0.3).view(2, 75)
    with torch.autocast("cuda", dtype=compute):
        loss = m.loss(tokens, targets)
        rows = m.out_norm(m(tokens)).detach()
    loss.backward()
    assert rows.dtype == torch.float32 and loss.dtype == torch.float32
    assert all(p.grad.dtype == dtype and p.grad.isfinite().all() for p in m.parameters() if p.grad is not None) and m.embedding.grad is not None
    with torch.no_grad():
        assert torch.equal(loss.detach(), moda_amd.linear_cross_entropy(rows.to(dtype), m.embedding, targets))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=names)
@pytest.mark.parametrize("rotary", [True, False])
def test_tokens_are_their_rows(dtype, rotary):
    m = model(dtype, True, rotary=rotary)
    tokens, lens = words(36, 517, 5).view(3, 12), torch.tensor([12, 7, 1], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        assert torch.equal(m(tokens), m(m.embed(tokens)))
    out = []
    for as_rows in (False, True):
        cache = moda_amd.PagedKVCache(2, 12, 16, 2, 16, dtype, "cuda", batch=3)
        for b in range(3):
            cache.reserve(b, 40)
        give = m.embed if as_rows else (lambda t: t)
        y = m.prefill(give(tokens), cache, lens)
        last = y[torch.arange(3), lens.long() - 1]
        step = m.decode(give(tokens[:, :1]), cache)
        nll = m.nll(step, tokens[:, 1:2])
        out.append((last, step, nll, cache.past.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*out)) and out[0][2].shape == (3, 1)


def test_next_words_are_scored_as_in_the_whole_sequence():
    """The likelihood of a sequence token by token from a cache and in one pass: rows that differ by what their attention rounds."""
    m = model(torch.float32, True)
    tokens = words(30, 517, 6).view(1, 30)
    with torch.no_grad():
        whole = m.nll(m(tokens[:, :-1]), tokens[:, 1:])
        cache = moda_amd.PagedKVCache(2, 4, 16, 2, 16, torch.float32, "cuda")
        cache.reserve(0, 30)
        parts = [m.nll(m.prefill(tokens[:, :9], cache), tokens[:, 1:10])]
        parts += [m.nll(m.decode(tokens[:, i:i + 1], cache), tokens[:, i + 1:i + 2]) for i in range(9, 29)]
        y = m.out_norm(m(tokens[:, :-1])).double()
    # Rows behind the norm have a length of sqrt(64); fp32 blocks of some thousand operations a row leave them within 2^-24 * 2^10 of that, a logit
    # within that times the longest word's row, and a loss within twice a logit.
    bound = 2 * y.norm(dim=-1).max() * m.embedding.double().norm(dim=-1).max() * 2.0 ** -14
    assert bool(((torch.cat(parts, 1).double() - whole.double()).abs() <= bound).all())


def test_captured_generation_step():
    """embed, decode and nll in one graph, replayed as the cache grows, with the program's own work between the replays."""
    m = model(torch.bfloat16, False)
    tokens = words(24, 517, 7).view(2, 12)

    def fresh():
        cache = moda_amd.PagedKVCache(2, 6, 16, 2, 16, torch.bfloat16, "cuda", batch=2)
        for b in range(2):
            cache.reserve(b, 40)
        m.prefill(tokens[:, :4], cache)
        return cache

    token, target = tokens[:, :1].clone(), tokens[:, 1:2].clone()
    eager, captured = fresh(), fresh()

    def step(cache):
        with torch.no_grad():
            y = m.decode(token, cache)
            return y, m.nll(y, target)

    step(fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(captured)
    for i in range(4, 10):
        token.copy_(tokens[:, i:i + 1])
        target.copy_(tokens[:, i + 1:i + 2])
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
