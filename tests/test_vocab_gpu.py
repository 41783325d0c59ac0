"""Token embedding and the cross entropy over a vocabulary against their definitions in 64 bits, on one MI355X.

Tolerances are bounds on each element, from the roundings that a kernel makes: u = eps / 2 of the tensors' type for a result (and, in the
backward pass of the cross entropy, for the gradient of a logit), 2^-24 for an fp32 operation, of which a sum of n terms has n."""
import contextlib
import math

import pytest
import torch

import moda_amd

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
F = 2.0 ** -24
NAME = {torch.bfloat16: "bf16", torch.float16: "fp16", torch.float32: "fp32"}
names = lambda d: NAME.get(d, str(d))  # noqa: E731


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance of the smallest values: what rounding takes where they lose bits."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isfinite(), want.isfinite()), what
    over = ((got - want).abs() - bound).nan_to_num(-1.0)
    assert bool((over <= 0).all()), f"{what}: {over.max().item():.3g} over its bound at {divmod(over.argmax().item(), max(1, got.shape[-1] if got.dim() else 1))}"


def rand(*shape, dtype, seed, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def words(n, vocab, seed, none=0.0, hot=0.0):
    """n tokens, a share of them no word, a share of them the same one."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, vocab, (n,), generator=g)
    u = torch.rand(n, generator=g)
    t[u < hot] = vocab // 3
    outside = torch.tensor([-1, vocab, -100, vocab + 12345, -(1 << 31)])
    bad = torch.rand(n, generator=g) < none
    t[bad] = outside[torch.randint(0, 5, (n,), generator=g)][bad]
    return t.cuda()


# ------------------------------------------------------------------------------------------------------------------
# embedding
# ------------------------------------------------------------------------------------------------------------------


def embed_reference(t, w, scale):
    live = (t >= 0) & (t < w.shape[0])
    y = w.double()[t.clamp(0, w.shape[0] - 1).long()] * scale
    return y * live[..., None]


def grad_reference(t, dy, vocab, scale):
    """The sum of a word's rows, and the bound of its fp32 sum."""
    t, dy = t.reshape(-1).long(), dy.double().reshape(-1, dy.shape[-1])
    live = (t >= 0) & (t < vocab)
    dw = torch.zeros(vocab, dy.shape[-1], dtype=torch.float64, device="cuda").index_add_(0, t[live], dy[live])
    size = torch.zeros_like(dw).index_add_(0, t[live], dy[live].abs())
    count = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, t[live], torch.ones_like(t[live], dtype=torch.float64))
    return dw * scale, size * abs(scale) * (count[:, None] + 1) * F


EMBED = [  # tokens, vocabulary, width, share that is no word, share that is one word
    (1, 1, 1, 0, 0), (1, 32000, 2048, 0, 0), (5, 7, 3, 0.3, 0), (33, 10, 64, 0, 0.5), (32, 4, 8, 0, 1), (64, 3, 16, 0, 1), (97, 3, 24, 0, 1),
    (1000, 1, 40, 0.1, 0), (3063, 50257, 384, 0.3, 0), (4097, 300, 129, 0.05, 0.2), (1025, 513, 4100, 0, 0.9), (9000, 40, 72, 0.2, 0.4),
    (140000, 262145, 8, 0.1, 0.1), (600, 1 << 19, 8, 1.0, 0),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n,vocab,width,none,hot", EMBED)
def test_embedding(dtype, n, vocab, width, none, hot):
    w, t = rand(vocab, width, dtype=dtype, seed=1), words(n, vocab, 2, none, hot)
    dy = rand(n, width, dtype=dtype, seed=3)
    for scale in (1.0, 0.37):
        w.requires_grad_()
        y = moda_amd.embed_tokens(t, w, scale)
        (dw,) = torch.autograd.grad(y, w, dy)
        want = embed_reference(t, w.detach(), scale)
        # the scale as fp32, the product, the result
        within(y.detach(), want, want.abs() * (half_step(dtype) * (scale != 1) + 3 * F * (scale != 1)) + smallest(dtype), "rows")
        want, sums = grad_reference(t, dy, vocab, scale)
        within(dw, want, want.abs() * (half_step(dtype) + 3 * F) + sums * (1 + half_step(dtype)) + smallest(dtype), "gradient")


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_embedding_layouts(dtype):
    base = rand(50, 80, dtype=dtype, seed=5)
    t = words(60, 50, 6, 0.2).view(3, 4, 5)
    for w in (base[:, 3:67], base[::2], base[:, ::2], base.t().contiguous().t(), base[:, :64], base[7:8].expand(50, 80)):
        for tokens in (t, t.clamp(-5, 100).int(), t.transpose(0, 2), t[:, ::2]):
            assert torch.equal(moda_amd.embed_tokens(tokens, w), embed_reference(tokens, w, 1.0).to(dtype))
    dy = rand(3, 4, 5, 160, dtype=dtype, seed=7)
    for d in (dy[..., :64], dy[..., 5:70], dy[..., ::2], dy[..., :1].expand(3, 4, 5, 24)):
        want, sums = grad_reference(t, d, 50, 1.0)
        within(moda_amd.embed_tokens_bwd(t, d, 50), want, want.abs() * half_step(dtype) + sums * 1.01 + smallest(dtype), "gradient")


def test_embedding_empty_and_special_values():
    w = rand(10, 16, dtype=torch.bfloat16, seed=8)
    assert moda_amd.embed_tokens(torch.zeros(0, 3, dtype=torch.long, device="cuda"), w).shape == (0, 3, 16)
    none = moda_amd.embed_tokens_bwd(torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 16, device="cuda"), 7)
    assert none.shape == (7, 16) and not none.any()
    w[3], w[4] = math.nan, math.inf
    y = moda_amd.embed_tokens(torch.tensor([3, -1, 4, 10, 5], device="cuda"), w)
    assert y[0].isnan().all() and y[2].isposinf().all() and not y[1].any() and not y[3].any() and torch.equal(y[4], w[5])
    dy = torch.ones(5, 16, device="cuda")
    dy[1], dy[3] = math.nan, math.inf  # rows of no word
    dw = moda_amd.embed_tokens_bwd(torch.tensor([3, -1, 4, 10, 3], device="cuda"), dy, 10)
    assert torch.equal(dw.sum(1), torch.tensor([0, 0, 0, 32.0, 16, 0, 0, 0, 0, 0], device="cuda"))


def test_embedding_twice_differentiable():
    w, t = rand(9, 24, dtype=torch.float32, seed=9).requires_grad_(), words(40, 9, 10, 0.2)
    dy = rand(40, 24, dtype=torch.float32, seed=11).requires_grad_()
    y = moda_amd.embed_tokens(t, w, 2.0)
    (dw,) = torch.autograd.grad(y, w, dy, create_graph=True)
    u = rand(9, 24, dtype=torch.float32, seed=12)
    (ddy,) = torch.autograd.grad(dw, dy, u)
    assert torch.equal(ddy, moda_amd.embed_tokens(t, u, 2.0))


# ------------------------------------------------------------------------------------------------------------------
# cross entropy
# ------------------------------------------------------------------------------------------------------------------


def loss_reference(x, w, t, scale, ignore_index, reduction, g=None):
    """loss, lse (base 2), dx, dw in 64 bits, and a bound for each."""
    dtype, shape = x.dtype, t.shape
    V, C = w.shape
    x, w, t = x.detach().double().reshape(-1, C), w.detach().double(), t.reshape(-1).long()
    live = ((t != ignore_index) & (t >= 0) & (t < V)).nonzero()[:, 0]
    N, n = t.numel(), live.numel()
    xl, tl, at = x[live], t[live], torch.arange(n, device="cuda")
    z = scale * xl @ w.T
    # a logit: its sum's terms (fp32: six products for each, and those left out), the scale in base 2
    terms = (C + 8) if dtype != torch.float32 else 2 * C + 16
    dz_bound = (abs(scale) * xl.abs() @ w.abs().T) * terms * F + z.abs() * 4 * F
    lse = torch.logsumexp(z, -1)
    loss = lse - z[at, tl]
    worst = dz_bound.amax(-1) if n else dz_bound.new_zeros(0)
    # exponentials (an ulp, and the rounding of an argument of up to log V that counts), sums by lane, tile and across tiles, the logarithm
    lse_bound = worst + (2 + math.log(V) + 64 + V / 128 + 8 + 8 * lse.abs()) * F
    loss_bound = lse_bound + worst + 8 * (loss.abs() + lse.abs()) * F
    rows, rows_bound, lse2, lse2_bound = (torch.zeros(N, dtype=torch.float64, device="cuda") for _ in range(4))
    rows[live], rows_bound[live], lse2[live] = loss, loss_bound, lse / math.log(2)
    lse2_bound[live] = lse_bound / math.log(2)
    out = {"lse": (lse2.view(shape), lse2_bound.view(shape))}
    share = 1.0 if reduction != "mean" else 1.0 / max(1, n)
    if reduction == "none":
        out["loss"] = rows.view(shape), rows_bound.view(shape)
    else:
        out["loss"] = rows.sum() * share, rows_bound.sum() * share + rows.sum().abs() * share * 2 * F
    if g is None:
        return out
    gl = (g.double().reshape(-1)[live] if reduction == "none" else g.double().expand(n) * share)[:, None]
    p = (z - lse[:, None]).exp()
    dz = gl * p
    # the hardware's exponential is zero where fp32 would have lost bits: below 2^-126
    dz_err = dz.abs() * ((dz_bound + lse_bound[:, None]) * 1.01 + 8 * F) + gl.abs() * 2.0 ** -126
    dz[at, tl] -= gl[:, 0]
    dz_err += dz.abs() * 4 * F
    if dtype != torch.float32:
        dz_err += dz.abs() * half_step(dtype)
        if dtype == torch.float16:  # kept 2^14 times as large, relative to the largest upstream gradient
            dz_err += smallest(dtype) * 2.0 ** -13 * gl.abs().max() if n else 0
    drop = 4 * F if dtype == torch.float32 else 0.0
    dx, dx_bound = torch.zeros_like(x), torch.zeros_like(x)
    dx[live] = scale * dz @ w
    dx_bound[live] = abs(scale) * (dz_err @ w.abs() + (V * F + drop) * 1.01 * dz.abs() @ w.abs())
    dw = scale * dz.T @ xl
    dw_bound = abs(scale) * (dz_err.T @ xl.abs() + (n * F + drop) * 1.01 * dz.abs().T @ xl.abs())
    for name, v, b in (("dx", dx, dx_bound), ("dw", dw, dw_bound)):
        out[name] = v, b * (1 + half_step(dtype)) + v.abs() * (half_step(dtype) + 3 * F) + smallest(dtype)
    out["dx"] = tuple(v.view(*shape, C) for v in out["dx"])
    return out


def check_loss(x, w, t, scale=1.0, ignore_index=-100, reduction="mean", seed=0):
    ref_x = x if x.dtype != torch.float32 else x
    g = rand(*(t.shape if reduction == "none" else ()), dtype=torch.float32, seed=seed + 50)
    ref = loss_reference(ref_x, w, t, scale, ignore_index, reduction, g)
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, scale, ignore_index, reduction)
    within(lse, *ref["lse"], "lse")
    within(loss, *ref["loss"], "loss")
    xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
    again = moda_amd.linear_cross_entropy(xg, wg, t, scale, ignore_index, reduction)
    assert torch.equal(again.detach(), loss)
    dx, dw = torch.autograd.grad(again, (xg, wg), g)
    within(dx, *ref["dx"], "dx")
    within(dw, *ref["dw"], "dw")
    return loss, dx, dw


LOSS = [  # rows, vocabulary, width
    (1, 1, 1), (1, 300, 64), (3, 17, 8), (31, 129, 24), (33, 257, 72), (128, 640, 64), (129, 1000, 40), (130, 513, 130), (257, 255, 257),
    (300, 5000, 256), (7, 40000, 64), (1000, 33, 520), (600, 700, 1024),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n,vocab,width", LOSS)
def test_loss(dtype, n, vocab, width):
    x, w = rand(n, width, dtype=dtype, seed=n), rand(vocab, width, dtype=dtype, seed=vocab, std=2 * width ** -0.5)
    for k, (reduction, none, scale) in enumerate([("mean", 0.0, 1.0), ("none", 0.4, 0.7), ("sum", 0.2, -3.0)]):
        check_loss(x, w, words(n, vocab, k, none), scale, reduction=reduction, seed=k)


# sizes of several tiles (csrc/vocab.h: choose_tiling), whole and split over their summation axis; TILES has each of them for each of the products
@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n,vocab,width", [(700, 9000, 512), (1500, 5000, 264), (8200, 1100, 2056), (4100, 2100, 2056), (1500, 12000, 1032), (5003, 9001, 520),
                                           (20, 30000, 1024)])
def test_loss_by_tile(dtype, n, vocab, width):
    x, w = rand(n, width, dtype=dtype, seed=n), rand(vocab, width, dtype=dtype, seed=vocab, std=2 * width ** -0.5)
    check_loss(x, w, words(n, vocab, 1, 0.2))
    check_loss(x, w, words(n, vocab, 2, 0.7), 0.6, reduction="none")


TILES = [  # what test_vocab_plan_cpu.py holds to take each tile, the rows read in place or not, for each product, whole and in sums
    # up to 512 rows of 16 bits are read where they are
    (509, 4099, 1000), (250, 13000, 520), (80, 50257, 512), (512, 66000, 1032), (511, 4099, 136), (512, 4099, 136), (513, 4099, 136), (397, 20011, 40), (5, 1100, 40),
    # the rows' gradient as it leaves the registers and by sums, the weight's
    (8200, 33, 1000), (3001, 33, 1032), (8200, 33, 40), (12001, 700, 40), (20001, 129, 40), (2100, 1100, 40), (2100, 1100, 72), (4100, 4099, 72), (3000, 9001, 264),
    (8200, 129, 1032), (12000, 129, 2056), (1000, 33, 40), (1, 50257, 40), (1, 30000, 264), (513, 129, 2056),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n,vocab,width", TILES)
def test_loss_by_each_tile(dtype, n, vocab, width):
    """Rows and weight inside wider ones, on the 16-byte grid; some rows without a target, which hold anything."""
    x, w = rand(n, width + 24, dtype=dtype, seed=n)[:, 8:width + 8], rand(vocab, width + 16, dtype=dtype, seed=vocab, std=2 * width ** -0.5)[:, 16:]
    t = words(n, vocab, 1, 0.3)
    t[0] = vocab - 1
    loss, dx, dw = check_loss(x, w, t, 0.8, reduction="none")
    gone = (t < 0) | (t >= vocab)
    assert not loss[gone].any() and not dx[gone].any()
    x[gone] = math.nan
    again = check_loss(x, w, t, 0.8, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip((loss, dx, dw), again))


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_loss_layouts(dtype):
    base, wide = rand(2, 9, 10, 200, dtype=dtype, seed=20), rand(120, 200, dtype=dtype, seed=21, std=0.2)
    t = words(180, 60, 22, 0.2).view(2, 9, 10)
    for x, w in [(base[..., :64], wide[:60, :64]), (base[..., 3:67], wide[::2, 64:128]), (base[..., ::2], wide[:60, 5:105]),
                 (base[:, :, :, 8:9].expand(2, 9, 10, 40), wide[3:4, :40].expand(60, 40)), (base[..., :64], wide[:64, :60].t())]:
        check_loss(x, w, t, reduction="none")
        check_loss(x[:, ::3], w, t[:, ::3].int().clamp(-7, 1000), reduction="sum")
    check_loss(base[0, 0, 0, :64], wide[:60, :64], torch.tensor(5, device="cuda"), reduction="none")


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n", [40, 300])
def test_rows_without_a_target_are_not_read(dtype, n):
    x, w, t = rand(n, 64, dtype=dtype, seed=30), rand(90, 64, dtype=dtype, seed=31, std=0.3), words(n, 90, 32, 0.5)
    t[::7] = 11
    clean = check_loss(x, w, t, ignore_index=11)
    dirty = x.clone()
    gone = (t < 0) | (t >= 90) | (t == 11)
    dirty[gone] = torch.where(torch.arange(int(gone.sum()), device="cuda")[:, None] % 2 == 0, math.nan, -math.inf).to(dtype)
    xg, wg = dirty.requires_grad_(), w.detach().requires_grad_()
    loss = moda_amd.linear_cross_entropy(xg, wg, t, ignore_index=11)
    dx, dw = torch.autograd.grad(loss, (xg, wg))
    want = torch.autograd.grad(moda_amd.linear_cross_entropy(x.requires_grad_(), wg, t, ignore_index=11), (x, wg))
    assert torch.equal(loss.detach(), clean[0]) and torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and not dx[gone].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n", [1, 200])
def test_no_row_has_a_target(dtype, n):
    x = torch.full((n, 40), math.nan, dtype=dtype, device="cuda").requires_grad_()
    w = rand(70, 40, dtype=dtype, seed=33).requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = moda_amd.linear_cross_entropy(x, w, torch.full((n,), -100, device="cuda"), reduction=reduction)
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert not loss.any() and not dx.any() and not dw.any()


def test_empty():
    x, w = torch.zeros(0, 16, device="cuda", dtype=torch.bfloat16).requires_grad_(), rand(20, 16, dtype=torch.bfloat16, seed=34).requires_grad_()
    t = torch.zeros(0, dtype=torch.long, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = moda_amd.linear_cross_entropy(x, w, t, reduction=reduction)
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert loss.numel() == (0 if reduction == "none" else 1) and not loss.any() and dx.shape == (0, 16) and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_what_is_not_finite_stays_in_its_rows(dtype):
    x, w, t = rand(150, 64, dtype=dtype, seed=35), rand(300, 64, dtype=dtype, seed=36, std=0.3), words(150, 300, 37)
    clean = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    x[3, 5], x[70, 1] = math.nan, math.inf
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    keep = torch.ones(150, dtype=torch.bool, device="cuda")
    keep[3] = keep[70] = False
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep]) and loss[~keep].isnan().all()
    dx, _ = moda_amd.linear_cross_entropy_bwd(x, w, t, lse, torch.ones(150, device="cuda"), reduction="none")
    assert dx[keep].isfinite().all() and dx[~keep].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("n,vocab,width", [(1, 300, 64), (150, 300, 64), (700, 9000, 512), (1500, 5000, 264), (40, 300000, 1024)])
def test_words_that_a_weight_rules_out(dtype, n, vocab, width):
    """A weight of minus infinity in a column where every row is positive: the word's logits are minus infinity, and all else is as without the word."""
    x, w = rand(n, width, dtype=dtype, seed=n), rand(vocab, width, dtype=dtype, seed=vocab, std=2 * width ** -0.5)
    x[:, 5] = x[:, 5].abs() + 0.1
    gone = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    gone[::7] = gone[-1] = True
    kept = (~gone).nonzero()[:, 0]
    place = words(n, kept.numel(), 3, 0.2)  # targets among the words that are left
    t = torch.where((place >= 0) & (place < kept.numel()), kept[place.clamp(0, kept.numel() - 1)], -100)
    left = w[kept]
    w[gone, 5] = -math.inf
    ref = loss_reference(x, left, torch.where(t < 0, -100, place), 1.0, -100, "none", torch.ones(n, device="cuda"))
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    within(loss, *ref["loss"], "loss")
    within(lse, *ref["lse"], "lse")
    dx, dw = moda_amd.linear_cross_entropy_bwd(x, w, t, lse, torch.ones(n, device="cuda"), reduction="none")
    assert not dw[gone].any()
    within(dw[kept], *ref["dw"], "dw")
    # the probability of a word that is ruled out is zero, and so is what its weights add, but for the infinite one: zero times that is NaN
    other = torch.arange(width, device="cuda") != 5
    within(dx[:, other], *(v[:, other] for v in ref["dx"]), "dx")
    assert dx[t >= 0, 5].isnan().all() and not dx[t < 0].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_infinite_products_keep_their_sign(dtype):
    """A row and a weight that meet at an infinite element: what is left of the row's log sum says which way each logit went."""
    x, w = rand(6, 64, dtype=dtype, seed=33), rand(40, 64, dtype=dtype, seed=34, std=0.3)
    t = torch.zeros(6, dtype=torch.long, device="cuda")
    w[:, 7] = -w[:, 7].abs() - 0.125  # (away from zero, where rounding takes an element apart)
    x[0, 7], x[1, 7], x[2, 7], x[3, 7] = math.inf, -math.inf, math.nan, 0.0
    z = x.double() @ w.double().T
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    want = torch.logsumexp(z, -1) - z[:, 0]  # all minus infinity, all infinite, NaN: no number; the others are their own
    assert torch.equal(loss.isnan(), want.isnan()) and loss[3:].isfinite().all() and loss[:3].isnan().all()
    w[20:, 7] = 0.0
    w[:20, 7] = -math.inf
    x[:, 7] = x[:, 7].nan_to_num(1.0, 1.0, 1.0).abs() + 0.5
    t += 30
    assert moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")[0].isfinite().all()
    x[0, 7] = -1.0  # of infinite logits the loss is no number
    assert moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")[0].isnan().tolist() == [True] + [False] * 5


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
def test_large_logits(dtype):
    """Logits of some hundreds: the likeliest word has all of the sum, and exponentials of the others leave fp32's range."""
    x, w, t = rand(140, 64, dtype=dtype, seed=38, std=8.0), rand(500, 64, dtype=dtype, seed=39, std=6.0), words(140, 500, 40)
    t[:70] = (x.double() @ w.double().T).argmax(-1)[:70]
    check_loss(x, w, t, reduction="none")


def test_upstream_gradients_far_apart_fp16():
    """The largest one sets the scale that dz is kept at; rows far below it lose bits relative to theirs alone."""
    x, w, t = rand(200, 64, dtype=torch.float16, seed=41), rand(400, 64, dtype=torch.float16, seed=42, std=0.3), words(200, 400, 43)
    for most in (2.0 ** -12, 1.0, 2.0 ** 9):
        g = torch.full((200,), most, device="cuda")
        g[::2] *= 2.0 ** -8
        ref = loss_reference(x, w, t, 1.0, -100, "none", g)
        _, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
        dx, dw = moda_amd.linear_cross_entropy_bwd(x, w, t, lse, g, reduction="none")
        within(dx, *ref["dx"], "dx")
        within(dw, *ref["dw"], "dw")


@pytest.mark.parametrize("dtype", DTYPES, ids=names)
@pytest.mark.parametrize("apart", [2.0 ** -12, 2.0 ** -14])
def test_small_upstream_gradients_keep_their_bits(dtype, apart):
    """Gradients of logits of 2^-26 of the largest upstream gradient and above have all of their bits, in fp16 too: rows far below the largest one are held
    to the bound that they would have in a call of their own."""
    x, w, t = rand(200, 64, dtype=dtype, seed=41), rand(400, 64, dtype=dtype, seed=42, std=0.03), words(200, 400, 43)
    g = torch.ones(200, device="cuda")
    small = torch.arange(0, 200, 2, device="cuda")
    g[small] *= apart
    _, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    dx, _ = moda_amd.linear_cross_entropy_bwd(x, w, t, lse, g, reduction="none")
    assert (x.double() @ w.double().T).softmax(-1).min() > 2.0 ** -12
    within(dx[small], *loss_reference(x[small], w, t[small], 1.0, -100, "none", g[small])["dx"], "dx")


@pytest.mark.parametrize("dtype,n,vocab,width", [(torch.bfloat16, 20000, 60000, 16), (torch.float32, 40, 300000, 1024), (torch.bfloat16, 17000, 50, 24),
                                                 (torch.float16, 17000, 3000, 72)], ids=str)
def test_many_rows_and_words(dtype, n, vocab, width):
    """More rows than a workgroup counts by itself; a vocabulary in pieces (of the logits' gradient, of the weight that is laid out anew)."""
    x, w = rand(n, width, dtype=dtype, seed=44), rand(vocab, width, dtype=dtype, seed=45, std=width ** -0.5)
    check_loss(x, w, words(n, vocab, 46, 0.3), reduction="mean")


@pytest.mark.parametrize("dtype,n,vocab,width", [(torch.bfloat16, 21, (1 << 22) + 777, 8), (torch.float16, 40, (1 << 21) + 1, 20), (torch.float32, 9, 600001, 1024)], ids=str)
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_statistics_of_several_pieces(dtype, n, vocab, width, reduction):
    """Three and more pieces of the vocabulary in the forward pass, the last of them short; targets at their borders; words whose logits are minus
    infinity throughout a piece, and rows whose largest logits are in the first or in the last one."""
    x, w = rand(n, width, dtype=dtype, seed=n), rand(vocab, width, dtype=dtype, seed=vocab, std=width ** -0.5)
    x[:, 3] = x[:, 3].abs() + 0.5
    w[100] = x[1] * 4 / x[1].float().norm()
    w[-1] = x[2] * 4 / x[2].float().norm()
    t = words(n, vocab, 46, 0.2)
    t[:6] = torch.tensor([0, vocab - 1, vocab - 1, 1 << 20, (1 << 21) - 1, vocab // 2], device="cuda")
    ref = loss_reference(x, w, t, 1.0, -100, reduction)
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction=reduction)
    within(lse, *ref["lse"], "lse")
    within(loss, *ref["loss"], "loss")
    # all words of the first half, whole pieces among them, ruled out
    half = vocab // 2
    w[:half, 3] = -math.inf
    t[t < half] = -100
    ref = loss_reference(x, w[half:], torch.where(t >= 0, t - half, -100), 1.0, -100, reduction)
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction=reduction)
    within(lse, *ref["lse"], "lse")
    within(loss, *ref["loss"], "loss")


@pytest.mark.parametrize("what", ["x", "w"])
def test_only_one_gradient(what):
    x, w, t = rand(200, 64, dtype=torch.bfloat16, seed=47), rand(600, 64, dtype=torch.bfloat16, seed=48), words(200, 600, 49, 0.1)
    both = [a.requires_grad_() for a in (x.clone(), w.clone())]
    want = torch.autograd.grad(moda_amd.linear_cross_entropy(*both, t), both)
    (x if what == "x" else w).requires_grad_()
    moda_amd.linear_cross_entropy(x, w, t).backward()
    assert torch.equal(x.grad if what == "x" else w.grad, want[what == "w"]) and (w if what == "x" else x).grad is None


def test_gradients_against_differences():
    """Along a direction d with |d x w| of the order of one: the difference quotient is off by e^2 / 6 times the third derivative, at most
    the cube of the logits' change, and by the losses' own roundings over e."""
    x, w, t = rand(20, 16, dtype=torch.float32, seed=60), rand(50, 16, dtype=torch.float32, seed=61, std=0.3), words(20, 50, 62, 0.1)
    for reduction in ("mean", "sum"):
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        dx, dw = torch.autograd.grad(moda_amd.linear_cross_entropy(xg, wg, t, reduction=reduction), (xg, wg))
        rows = 1 if reduction == "mean" else 20
        for k, (ux, uw) in enumerate([(rand(20, 16, dtype=torch.float32, seed=63, std=0.3), 0), (0, rand(50, 16, dtype=torch.float32, seed=64, std=0.3))]):
            e = 2.0 ** -5
            f = [moda_amd.linear_cross_entropy(x + s * e * ux, w + s * e * uw, t, reduction=reduction).double() for s in (1, -1)]
            slope = (ux.double() * dx.double()).sum() if k == 0 else (uw.double() * dw.double()).sum()
            change = ((ux.double() @ w.double().T) if k == 0 else (x.double() @ uw.double().T)).abs().max()
            assert abs((f[0] - f[1]) / (2 * e) - slope) <= rows * (e * e / 6 * 8 * change ** 3 + 64 * F * 10 / e)


def test_the_same_bits_every_time():
    x, w, t = rand(700, 512, dtype=torch.bfloat16, seed=65), rand(3001, 512, dtype=torch.bfloat16, seed=66, std=0.05), words(700, 3001, 67, 0.2, 0.3)
    def once():
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = moda_amd.linear_cross_entropy(xg, wg, t)
        return [loss.detach(), *torch.autograd.grad(loss, (xg, wg)), moda_amd.embed_tokens_bwd(t, x, 3001)]
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_captured_calls_follow_their_inputs():
    """One graph with both ends and their gradients, replayed with other tokens and rows, eager work between the replays."""
    w = rand(900, 128, dtype=torch.bfloat16, seed=70, std=0.1)
    t, x = words(400, 900, 71, 0.2), rand(400, 128, dtype=torch.bfloat16, seed=72)

    def step():
        y = moda_amd.embed_tokens(t, w, 2.0)
        loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t)
        one = torch.ones((), device="cuda")
        return [y, moda_amd.embed_tokens_bwd(t, x, 900, 2.0), loss, *moda_amd.linear_cross_entropy_bwd(x, w, t, lse, one)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        t.copy_(words(400, 900, 80 + k, 0.2 * k))
        x.copy_(rand(400, 128, dtype=torch.bfloat16, seed=90 + k))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_captured_backward():
    """Both ends around torch's own sum, one weight for both, with autograd's engine in the capture; leaves are made in the captured step."""
    w = rand(900, 128, dtype=torch.bfloat16, seed=73, std=0.1)
    t, x = words(300, 900, 74, 0.2), rand(300, 128, dtype=torch.bfloat16, seed=75)

    def step():
        xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = moda_amd.linear_cross_entropy(xg + moda_amd.embed_tokens(t, wg, 2.0), wg, t)
        return [loss.detach(), *torch.autograd.grad(loss, (xg, wg))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        t.copy_(words(300, 900, 80 + k, 0.2 * k))
        x.copy_(rand(300, 128, dtype=torch.bfloat16, seed=90 + k))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_compiled_autograd():
    """Compiled autograd runs the nodes from a graph of its own: the same bits."""
    import torch._dynamo.compiled_autograd as compiled

    x, w, t = rand(40, 64, dtype=torch.bfloat16, seed=76), rand(90, 64, dtype=torch.bfloat16, seed=77, std=0.1), words(40, 90, 78, 0.2)
    grads = []
    for k in range(3):
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = moda_amd.linear_cross_entropy(xg + moda_amd.embed_tokens(t, wg, 2.0), wg, t, reduction="sum")
        with compiled._enable(lambda graph: graph) if k else contextlib.nullcontext():
            loss.backward()
        grads.append((xg.grad, wg.grad))
    assert all(torch.equal(a, b) for g in grads[1:] for a, b in zip(grads[0], g))


def test_calls_on_two_streams():
    x = [rand(500, 256, dtype=torch.bfloat16, seed=100 + i) for i in range(2)]
    w, t = rand(2000, 256, dtype=torch.bfloat16, seed=102, std=0.1), [words(500, 2000, 103 + i, 0.1) for i in range(2)]

    def step(i):
        loss, lse = moda_amd.linear_cross_entropy_fwd(x[i], w, t[i])
        return [loss, *moda_amd.linear_cross_entropy_bwd(x[i], w, t[i], lse, torch.ones((), device="cuda")), moda_amd.embed_tokens_bwd(t[i], x[i], 2000)]

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))


def test_second_derivative_is_refused():
    x, w = rand(4, 16, dtype=torch.float32, seed=110).requires_grad_(), rand(9, 16, dtype=torch.float32, seed=111).requires_grad_()
    loss = moda_amd.linear_cross_entropy(x, w, words(4, 9, 112))
    (dx,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()


def test_changed_inputs_are_noticed():
    x, w, t = rand(4, 16, dtype=torch.float32, seed=113).requires_grad_(), rand(9, 16, dtype=torch.float32, seed=114), words(4, 9, 115)
    for a in (w, t):
        loss = moda_amd.linear_cross_entropy(x, w, t)
        a.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_traced_calls():
    w, t = rand(60, 32, dtype=torch.float32, seed=116), words(10, 60, 117, 0.1)

    def f(w, x, t):
        return moda_amd.linear_cross_entropy(x + moda_amd.embed_tokens(t, w, 0.5), w, t)

    x = rand(10, 32, dtype=torch.float32, seed=118)
    traced = torch.jit.trace(f, (w, x, t), check_trace=False)
    other = rand(10, 32, dtype=torch.float32, seed=119)
    assert torch.equal(traced(w, other, t), f(w, other, t))


def test_forward_mode_is_refused():
    x, w, t = rand(4, 16, dtype=torch.float32, seed=120), rand(9, 16, dtype=torch.float32, seed=121), words(4, 9, 122)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: moda_amd.embed_tokens(t, dual), lambda: moda_amd.linear_cross_entropy(x, dual, t), lambda: moda_amd.linear_cross_entropy(dual[:4], w, t)):
            with pytest.raises(RuntimeError):
                call()


def test_derivatives_are_not_dropped():
    """The two passes by themselves record nothing: what a caller could hope to differentiate is refused, but for rows and weight, which are constants."""
    x, w, t = rand(4, 16, dtype=torch.float32, seed=120), rand(9, 16, dtype=torch.float32, seed=121), words(4, 9, 122)
    one = torch.ones((), device="cuda")
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss, lse = moda_amd.linear_cross_entropy_fwd(xg, wg, t)
    assert not loss.requires_grad and not lse.requires_grad
    assert not any(g.requires_grad for g in moda_amd.linear_cross_entropy_bwd(xg, wg, t, lse, one))
    for late in ((lse.clone().requires_grad_(), one), (lse, one.clone().requires_grad_())):
        with pytest.raises(AssertionError, match="no backward pass"):
            moda_amd.linear_cross_entropy_bwd(x, w, t, *late)
        with torch.no_grad():
            moda_amd.linear_cross_entropy_bwd(x, w, t, *late)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda a: torch.autograd.forward_ad.make_dual(a, torch.ones_like(a))  # noqa: E731
        for call in (lambda: moda_amd.linear_cross_entropy_fwd(dual(x), w, t), lambda: moda_amd.linear_cross_entropy_fwd(x, dual(w), t),
                     lambda: moda_amd.linear_cross_entropy_bwd(dual(x), w, t, lse, one), lambda: moda_amd.linear_cross_entropy_bwd(x, dual(w), t, lse, one),
                     lambda: moda_amd.linear_cross_entropy_bwd(x, w, t, dual(lse), one), lambda: moda_amd.linear_cross_entropy_bwd(x, w, t, lse, dual(one))):
            with pytest.raises(AssertionError, match="tangent"):
                call()


def test_refusals():
    x, w, t = rand(4, 16, dtype=torch.bfloat16, seed=123), rand(9, 16, dtype=torch.bfloat16, seed=124), words(4, 9, 125)
    for call in (lambda: moda_amd.embed_tokens(t.float(), w), lambda: moda_amd.embed_tokens(t.cpu(), w), lambda: moda_amd.embed_tokens(t, w[0]),
                 lambda: moda_amd.embed_tokens(t, w, math.nan), lambda: moda_amd.embed_tokens(t, w[:0]), lambda: moda_amd.embed_tokens_bwd(t, x[:3], 9),
                 lambda: moda_amd.embed_tokens_bwd(t, x, 0), lambda: moda_amd.linear_cross_entropy(x[:, :8], w, t),
                 lambda: moda_amd.linear_cross_entropy(x, w, t[:3]), lambda: moda_amd.linear_cross_entropy(x, w, t.short()),
                 lambda: moda_amd.linear_cross_entropy(x, w, t, scale=math.inf), lambda: moda_amd.linear_cross_entropy(x, w.cpu().cuda()[:, None], t),
                 lambda: moda_amd.linear_cross_entropy_bwd(x, w, t, torch.zeros(3, device="cuda"), torch.ones((), device="cuda")),
                 lambda: moda_amd.linear_cross_entropy_bwd(x, w, t, torch.zeros(4, device="cuda"), torch.ones(4, device="cuda"))):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: moda_amd.linear_cross_entropy(x.float(), w, t), lambda: moda_amd.embed_tokens(t, w.double())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="reduction"):
        moda_amd.linear_cross_entropy(x, w, t, reduction="max")


def test_offsets_past_32_bits_embedding():
    vocab, width = (1 << 21) + 300, 1024
    w = torch.empty(vocab, width, dtype=torch.bfloat16, device="cuda").fill_(0.25)
    w[-40:] = rand(40, width, dtype=torch.bfloat16, seed=130)
    t = torch.cat([torch.arange(vocab - 40, vocab, device="cuda").repeat(3), torch.tensor([0, 7, vocab], device="cuda")])
    y = moda_amd.embed_tokens(t, w)
    assert torch.equal(y, embed_reference(t, w, 1.0).bfloat16())
    dy = rand(t.numel(), width, dtype=torch.bfloat16, seed=131)
    dw = moda_amd.embed_tokens_bwd(t, dy, vocab)
    want, sums = grad_reference(t - (vocab - 40), dy, 40, 1.0)
    within(dw[-40:], want, want.abs() * half_step(dy.dtype) + sums * 1.01, "gradient")
    assert torch.equal(dw[0], dy[-3]) and torch.equal(dw[7], dy[-2]) and int(dw.any(1).sum()) == 42


def test_offsets_past_32_bits_weight():
    vocab, width, n = (1 << 19) + 1000, 4104, 9
    w = torch.empty(vocab, width, dtype=torch.bfloat16, device="cuda").normal_(0.0, width ** -0.5, generator=torch.Generator("cuda").manual_seed(132))
    x = rand(n, width, dtype=torch.bfloat16, seed=133)
    t = torch.arange(vocab - n, vocab, device="cuda")
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    z = torch.cat([x.double() @ w[i:i + 65536].double().T for i in range(0, vocab, 65536)], 1)
    want = torch.logsumexp(z, -1)
    # as loss_reference's bounds, with |z| at most 8 and the sums of its terms at most width ** 0.5 times that
    bound = 2 * (width + 8) * F * (x.double().abs() @ w[-4096:].double().abs().T).max() * 2 + (64 + vocab / 128) * F
    within(loss, want - z[torch.arange(n), t], bound.expand(n), "loss")
    dx, dw = moda_amd.linear_cross_entropy_bwd(x, w, t, lse, torch.ones(n, device="cuda"), reduction="none")
    p = (z - want[:, None]).exp()
    p[torch.arange(n), t] -= 1
    for rows in (slice(0, 500), slice(vocab - 500, vocab)):
        size = p[:, rows].abs().T @ x.double().abs()
        within(dw[rows], p[:, rows].T @ x.double(), size * (2 * half_step(x.dtype) + 2 * bound + 64 * F) + smallest(x.dtype), "dw")
    want = sum(p[:, i:i + 65536] @ w[i:i + 65536].double() for i in range(0, vocab, 65536))
    size = sum(p[:, i:i + 65536].abs() @ w[i:i + 65536].double().abs() for i in range(0, vocab, 65536))
    within(dx, want, size * (2 * half_step(x.dtype) + 2 * bound + vocab * F), "dx")


def test_offsets_past_32_bits_rows():
    n, vocab, width = 270000, 40, 8192
    x = torch.empty(n, width, dtype=torch.bfloat16, device="cuda").normal_(0.0, 1.0, generator=torch.Generator("cuda").manual_seed(134))
    w, t = rand(vocab, width, dtype=torch.bfloat16, seed=135, std=width ** -0.5), words(n, vocab, 136, 0.1)
    loss, lse = moda_amd.linear_cross_entropy_fwd(x, w, t, reduction="none")
    dx, _ = moda_amd.linear_cross_entropy_bwd(x, w, t, lse, torch.ones(n, device="cuda"), reduction="none", need_dweight=False)
    for part in (slice(0, 300), slice(n - 300, n)):
        ref = loss_reference(x[part], w, t[part], 1.0, -100, "none", torch.ones(300, device="cuda"))
        within(loss[part], *ref["loss"], "loss")
        within(dx[part], *ref["dx"], "dx")
