"""Rotary positions, appending to a paged key/value cache and the attention over it, on the GPU against plain
implementations in 64 bits.

Tolerances, from the arithmetic.  u = half a unit in the last place of the output type relative to the value (bf16 2^-8, fp16
2^-11, fp32 2^-24).
  rotation: y = A (x0 cos - x1 sin).  The fraction of a turn is rounded to 2^-26 of a turn (the angle to 2^-23.3), sine and cosine
    to 2 units (2^-22.. of 1), the amplitude, both products and their sum to 2^-24 each: A (|x0| + |x1|) 2^-21 covers them;
    then one rounding of the result, u |y| (fp16 below 2^-14: 2^-25).
  attention: logits in base 2 are off by at most e = (D + 4) 2^-24 scale max |q| |k| log2(e) (a sum of D products, scale), a
    probability by the factor 2^e (1 + 2^-22), sums of n terms by n 2^-24; with probabilities rounded to the type (u) before
    they meet the values: (u + 2 e + n 2^-24 + 2^-20) sum p |v| in all, then one rounding u |o|.
    lse: e + n 2^-24 + 2^-22 max(1, |lse|).
"""
import itertools
import math

import pytest
import torch

import moda_amd

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TINY = {BF16: 0.0, FP16: 2.0 ** -25, FP32: 0.0}


def close(got, want, tol, what):
    """|got - want| <= tol element by element; NaN where and only where the reference has one, infinities equal."""
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~want.isfinite()
    assert torch.equal(got[odd].nan_to_num(7e300), want[odd].nan_to_num(7e300)), f"{what}: non-finite values differ"
    bad = ~((got - want).abs() <= tol) & ~odd
    if bad.any():
        i = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[tuple(i)]} for {want[tuple(i)]}, "
                             f"allowed {tol[tuple(i)]}")


# ------------------------------------------------------------------------------------------------------------------
# rotation
# ------------------------------------------------------------------------------------------------------------------


def rotation64(x, pos, rot, inverse=False):
    """x [..., rows, heads, D], pos [..., rows]: (rotated, sum of magnitudes of what each element is made of)."""
    x = x.detach().double().cpu()
    f = rot._host
    a = torch.remainder(pos.cpu().double()[..., None] * f, 1.0) * 2 * math.pi
    c, s = a.cos()[..., None, :] * rot.amplitude, a.sin()[..., None, :] * rot.amplitude * (-1 if inverse else 1)
    y, m = x.clone(), torch.zeros_like(x)
    R = rot.dim
    i0, i1 = (range(0, R, 2), range(1, R, 2)) if rot.interleaved else (range(R // 2), range(R // 2, R))
    i0, i1 = list(i0), list(i1)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    both = (x0.abs() + x1.abs()) * rot.amplitude
    m[..., i0], m[..., i1] = both, both
    return y, m


def check_rotated(got, x, pos, rot, what, inverse=False):
    want, m = rotation64(x, pos, rot, inverse)
    close(got, want, U[x.dtype] * want.abs() * (m > 0) + m * 2.0 ** -21 + TINY[x.dtype] * (m > 0), what)


ROTATIONS = [
    # dtype, B, T, Hq, H, G, D, R, interleaved, positions
    (BF16, 1, 1, 4, 4, 4, 128, 128, False, None),
    (BF16, 2, 33, 2, 2, 4, 128, 64, True, "far"),
    (FP16, 3, 17, 3, 3, 2, 64, 64, True, "batch"),
    (FP16, 1, 130, 1, 1, 1, 64, 16, False, "far"),
    (FP32, 2, 19, 6, 2, 1, 64, 32, True, "far"),
    (FP32, 1, 65, 1, 1, 8, 256, 256, False, "int32"),
    (BF16, 2, 9, 5, 5, 3, 80, 80, False, "batch"),
    (BF16, 1, 11, 2, 1, 1, 20, 10, False, None),      # rows off the 16-byte grid
    (FP16, 1, 12, 1, 3, 2, 64, 22, True, "negative"),  # pairs that are no whole vectors
    (FP32, 1, 5, 1, 1, 1, 6, 2, False, "far"),
    (BF16, 1, 3000, 4, 4, 4, 64, 64, False, None),
    (BF16, 1, 7, 16, 8, 1, 256, 128, True, "far"),
    (FP32, 1, 3, 1, 1, 1, 512, 512, False, None),      # as many pairs as there are lanes
    (BF16, 1, 2, 1, 1, 1, 510, 510, True, "int32"),    # the same element by element
    (BF16, 1, 70000, 4, 4, 4, 128, 128, False, None),  # more than the memory-side cache holds
]


def make_positions(kind, B, T, dev):
    g = torch.Generator().manual_seed(7)
    if kind is None:
        return None, torch.arange(T).expand(B, T)
    p = {"far": lambda: torch.randint(900000, 1100000, (T,), generator=g), "int32": lambda: torch.arange(5, 5 + T, dtype=torch.int32),
         "batch": lambda: torch.randint(0, 70000, (B, T), generator=g), "negative": lambda: torch.arange(-5, T - 5)}[kind]()
    return p.to(dev), p.expand(B, T)


@pytest.mark.parametrize("case", ROTATIONS, ids=str)
def test_rotation_and_its_gradient(case, gpu_device):
    dtype, B, T, Hq, H, G, D, R, inter, kind = case
    torch.manual_seed(1)
    rot = moda_amd.Rotary(R, interleaved=inter, scaling="by_parts" if R > 2 and kind == "far" else None, factor=8.0, original_length=4096)
    q = torch.randn(B, T * G, Hq, D).to(dtype).to(gpu_device).requires_grad_()
    k = torch.randn(B, T, H, D).to(dtype).to(gpu_device).requires_grad_()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    p, per_token = make_positions(kind, B, T, gpu_device)
    q1, k1 = moda_amd.apply_rotary(q, k, rot, positions=p, moda_group_num=G)
    gq, gk = torch.autograd.grad((q1, k1), (q, k), (dq, dk))
    rows = per_token.repeat_interleave(G, 1)
    check_rotated(q1, q, rows, rot, "q")
    check_rotated(k1, k, per_token, rot, "k")
    check_rotated(gq, dq, rows, rot, "dq", inverse=True)
    check_rotated(gk, dk, per_token, rot, "dk", inverse=True)


def test_rotation_scalings(gpu_device):
    x = torch.randn(1, 50, 2, 64, device=gpu_device)
    p = torch.arange(100000, 100050, device=gpu_device)
    for scaling, inter in itertools.product((None, "linear", "ntk", "by_parts"), (False, True)):
        rot = moda_amd.Rotary(48, interleaved=inter, scaling=scaling, factor=4.0, original_length=8192)
        check_rotated(moda_amd.apply_rotary(x, None, rot, positions=p)[0], x, p[None], rot, f"{scaling} {inter}")


def test_gradient_of_a_rotation_against_differences(gpu_device):
    torch.manual_seed(2)
    rot = moda_amd.Rotary(12, scaling="by_parts", factor=2.0, original_length=64)
    q, k = torch.randn(1, 4, 2, 16, device=gpu_device), torch.randn(1, 2, 1, 16, device=gpu_device)
    wq, wk = torch.randn_like(q), torch.randn_like(k)

    def loss(q, k):
        a, b = moda_amd.apply_rotary(q, k, rot, moda_group_num=2)
        return (a * wq).sum(dtype=torch.float64) + (b * wk).sum(dtype=torch.float64)

    q.requires_grad_(), k.requires_grad_()
    gq, gk = torch.autograd.grad(loss(q, k), (q, k))
    for x, g in ((q, gq), (k, gk)):
        d = torch.randn_like(x)
        step = 2.0 ** -2  # the map is linear: any step is exact but for the roundings of two sums of 48 products
        with torch.no_grad():
            args = [(q + step * d, k), (q - step * d, k)] if x is q else [(q, k + step * d), (q, k - step * d)]
            slope = (loss(*args[0]) - loss(*args[1])) / (2 * step)
        magnitude = (x.abs().sum() + d.abs().sum()) * 4 * 3
        assert abs(float(slope - (g * d).sum(dtype=torch.float64))) <= 2.0 ** -20 * float(magnitude) / step


def test_rotation_one_tensor_strides_broadcast_second_derivative(gpu_device):
    torch.manual_seed(3)
    rot = moda_amd.Rotary(32)
    base = torch.randn(2, 7, 5, 3, 40, device=gpu_device).to(BF16)
    x = base[:, :, 1:4, :, :].select(2, 1)                       # strided rows, 80-byte heads
    pos = torch.arange(7).expand(2, 7)
    check_rotated(moda_amd.apply_rotary(None, x, rot)[1], x, pos, rot, "strided")
    y = x.transpose(2, 3).contiguous().transpose(2, 3)           # inner stride other than 1: copied
    check_rotated(moda_amd.apply_rotary(y, None, rot)[0], y, pos, rot, "inner stride")
    leaf = torch.randn(1, 7, 1, 32, device=gpu_device, requires_grad=True)
    wide = leaf.expand(3, 7, 4, 32)
    out = moda_amd.apply_rotary(wide, None, rot)[0]
    check_rotated(out, wide, torch.arange(7).expand(3, 7), rot, "broadcast")
    w = torch.randn_like(out, requires_grad=True)
    (g,) = torch.autograd.grad(out, leaf, w, create_graph=True)
    back, m = rotation64(w, torch.arange(7).expand(3, 7), rot, inverse=True)
    close(g, back.sum((0, 2), keepdim=True), m.sum((0, 2), keepdim=True) * 2.0 ** -20, "gradient of a broadcast")
    (gg,) = torch.autograd.grad(g.sum(), w)                      # d/dw of sum R^T w: R applied to ones
    check_rotated(gg, torch.ones_like(w), torch.arange(7).expand(3, 7), rot, "second derivative")
    # one gradient of two, and none
    q, k = torch.randn(1, 7, 1, 32, device=gpu_device, requires_grad=True), torch.randn(1, 7, 1, 32, device=gpu_device, requires_grad=True)
    a, b = moda_amd.apply_rotary(q, k, rot)
    (gk,) = torch.autograd.grad(b.sum(), k)
    check_rotated(gk, torch.ones_like(k), torch.arange(7)[None], rot, "k alone", inverse=True)
    a, b = moda_amd.apply_rotary(q, k.detach(), rot)
    (gq,) = torch.autograd.grad(a.sum(), q)
    check_rotated(gq, torch.ones_like(q), torch.arange(7)[None], rot, "q alone", inverse=True)
    # a positions tensor that changes between the passes is noticed
    p = torch.arange(7, device=gpu_device)
    a, _ = moda_amd.apply_rotary(q, None, rot, positions=p)
    p.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        a.sum().backward()
    assert moda_amd.apply_rotary(torch.empty(0, 4, 2, 32, device=gpu_device), None, rot)[0].shape == (0, 4, 2, 32)


def test_rotation_traced(gpu_device):
    rot = moda_amd.Rotary(16)
    q, k = torch.randn(1, 8, 2, 16, device=gpu_device), torch.randn(1, 4, 2, 16, device=gpu_device)
    f = torch.jit.trace(lambda q, k: moda_amd.apply_rotary(q, k, rot, moda_group_num=2), (q, k), check_trace=False)
    q2, k2 = torch.randn_like(q), torch.randn_like(k)
    got, want = f(q2, k2), moda_amd.apply_rotary(q2, k2, rot, moda_group_num=2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------------------------------
# pages
# ------------------------------------------------------------------------------------------------------------------


class Cache:
    """Pages in a shuffled order, NaN wherever no token is; `layout` "heads": pages [n, H, P, D] seen as [n, P, H, D]."""

    def __init__(self, dev, dtype, B, H, D, Dv, P, past, new, layout="tokens", spare=2):
        lens = [p + n for p, n in zip(past, new)]
        need = [-(-x // P) for x in lens]
        n = sum(need) + spare
        g = torch.Generator().manual_seed(11)
        order = torch.randperm(n, generator=g).int().tolist()
        width = max(max(need), 1) + 1
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        for b in range(B):
            for i in range(need[b]):
                self.table[b, i] = order.pop()
        self.K = [torch.randn(x, H, D, generator=g).to(dtype) for x in lens]  # tokens of each sequence
        self.V = [torch.randn(x, H, Dv, generator=g).to(dtype) for x in lens]
        self.P, self.past = P, past
        shape = (n, P, H) if layout == "tokens" else (n, H, P)
        self.k, self.v = (torch.full((*shape, d), math.nan, dtype=dtype) for d in (D, Dv))
        if layout == "heads":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for b in range(B):
            for j in range(lens[b]):
                self.k[self.table[b, j // P], j % P], self.v[self.table[b, j // P], j % P] = self.K[b][j], self.V[b][j]
        self.k, self.v = (x.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if layout == "heads" else x.to(dev) for x in (self.k, self.v))
        self.table_dev, self.past_dev = self.table.to(dev), torch.tensor(past, dtype=torch.int32, device=dev)


def reference_attention(q, keys, values, scale):
    """q [rows, D], keys [n, D], values [n, Dv] in 64 bits -> o, lse (base 2), e, sum p |v|; what is not seen is not there."""
    if keys.shape[0] == 0:
        return torch.zeros(q.shape[0], values.shape[1], dtype=torch.float64), torch.full((q.shape[0],), -math.inf, dtype=torch.float64), \
            torch.zeros(q.shape[0], dtype=torch.float64), torch.zeros(q.shape[0], values.shape[1], dtype=torch.float64)
    s = q @ keys.T * (scale / math.log(2))
    lse = torch.logsumexp(s * math.log(2), -1) / math.log(2)
    p = torch.exp2(s - lse[:, None])
    e = (q.abs() @ keys.abs().T).amax(-1) * (scale / math.log(2)) * (q.shape[1] + 4) * 2.0 ** -24
    return p @ values, lse, e, p @ values.abs()


def check_attention(c, q, o, lse, T, G, H, new, scale, plain, depth=None, L=0, Lv=0, what=""):
    """depth: (kd, vd) [B, T*L, H, *] on the CPU; rows in float64 against what each sees."""
    B, dtype = q.shape[0], q.dtype
    q = q.detach().double().cpu()
    want, wl = torch.zeros(o.shape, dtype=torch.float64), torch.full(lse.shape, -math.inf, dtype=torch.float64)
    tol, tl = torch.zeros_like(want), torch.zeros_like(wl)
    for b in range(B):
        for t in range(min(new[b], T)):
            for h in range(H):
                keys, values = c.K[b][:c.past[b] + t + 1, h].double(), c.V[b][:c.past[b] + t + 1, h].double()
                if depth:
                    r = slice(t * L, t * L + Lv)
                    keys, values = torch.cat([keys, depth[0][b, r, h].double()]), torch.cat([values, depth[1][b, r, h].double()])
                at = (b, t, slice(h * G, h * G + G)) if plain else (b, slice(t * G, t * G + G), h)
                x, l, e, m = reference_attention(q[at], keys, values, scale)
                n = keys.shape[0]
                want[at], wl[at] = x, l
                tol[at] = U[dtype] * x.abs() + (U[dtype] + 2 * e[:, None] + n * 2.0 ** -24 + 2.0 ** -20) * m + TINY[dtype]
                tl[at] = e + n * 2.0 ** -24 + 2.0 ** -22 * l.abs().clamp(min=1)
    close(o, want, tol, what + " o")
    close(lse, wl, tl, what + " lse")


ATTEND = [
    # dtype, H, G, D, Dv, page, T, L, Lv, past, new (None: T each), layout
    (BF16, 4, 4, 128, 128, 16, 1, 24, 8, [100], None, "tokens"),
    (BF16, 1, 1, 64, 64, 16, 1, 0, 0, [0], None, "tokens"),                       # the first token of all
    (BF16, 2, 4, 128, 128, 16, 1, 0, 0, [0, 14, 15, 16, 30, 31, 32, 33, 127], None, "tokens"),
    (FP16, 2, 8, 64, 64, 32, 1, 33, 33, [62, 63, 64, 255, 256, 1], None, "heads"),
    (FP16, 3, 3, 80, 80, 1, 1, 5, 1, [40, 3], None, "tokens"),                    # a page a token
    (BF16, 1, 16, 256, 256, 64, 1, 2, 2, [200, 77], None, "tokens"),
    (BF16, 2, 17, 128, 128, 16, 1, 70, 70, [45, 300], None, "tokens"),            # more rows than one tile of rows
    (BF16, 1, 40, 192, 64, 128, 1, 3, 2, [129], None, "tokens"),
    (FP16, 2, 2, 24, 128, 16, 1, 1, 1, [33, 65], None, "heads"),
    (BF16, 1, 1, 8, 8, 8, 1, 1, 1, [9], None, "tokens"),
    (FP32, 2, 1, 64, 64, 16, 1, 4, 3, [33, 100, 0], None, "tokens"),
    (FP32, 1, 5, 128, 128, 32, 1, 0, 0, [70, 15], None, "heads"),
    (FP32, 1, 20, 256, 256, 4, 1, 9, 9, [13], None, "tokens"),
    (FP32, 2, 3, 12, 100, 16, 2, 2, 1, [17, 40], None, "tokens"),
    (BF16, 2, 4, 128, 128, 16, 5, 24, 23, [0, 11, 16, 60, 200], [5, 0, 3, 1, 5], "tokens"),  # drafted tokens, fewer for some
    (FP16, 1, 8, 64, 64, 32, 8, 12, 12, [30, 31, 0], None, "heads"),
    (BF16, 1, 3, 96, 96, 16, 13, 40, 3, [100, 5], [13, 2], "tokens"),
    (FP32, 1, 4, 64, 64, 16, 5, 8, 8, [30, 1], [4, 5], "tokens"),
    (FP16, 2, 8, 128, 128, 64, 16, 0, 0, [500], None, "tokens"),                  # 128 query rows a head
    (BF16, 2, 1, 64, 64, 16, 3, 100, 99, [20, 0, 7], [0, 0, 0], "tokens"),        # nobody has a new token
    (BF16, 2, 4, 128, 128, 16, 1, 24, 12, [2500, 1, 900, 0, 63, 64, 4000], None, "tokens"),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
@pytest.mark.parametrize("plain", [False, True], ids=["folded", "plain"])
def test_attention_over_pages(case, plain, gpu_device):
    dtype, H, G, D, Dv, P, T, L, Lv, past, new, layout = case
    if plain:
        L = Lv = 0
    torch.manual_seed(5)
    B = len(past)
    c = Cache(gpu_device, dtype, B, H, D, Dv, P, past, new or [T] * B, layout)
    q = torch.randn((B, T, H * G, D) if plain else (B, T * G, H, D)).to(dtype).to(gpu_device)
    new_dev = None if new is None else torch.tensor(new, dtype=torch.int32, device=gpu_device)
    scale, depth = D ** -0.5, None
    if plain:
        o, lse = moda_amd.paged_attn_fwd(q, c.k, c.v, c.table_dev, c.past_dev, new_lens=new_dev)
    else:
        if L:
            kd, vd = torch.full((B, T, L, H, D), math.nan, dtype=dtype), torch.full((B, T, L, H, Dv), math.nan, dtype=dtype)
            kd[:, :, :Lv], vd[:, :, :Lv] = torch.randn(B, T, Lv, H, D).to(dtype), torch.randn(B, T, Lv, H, Dv).to(dtype)
            depth = kd.view(B, T * L, H, D), vd.view(B, T * L, H, Dv)
        dev = [x.to(gpu_device) for x in depth] if depth else [None, None]
        o, lse = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, new_lens=new_dev, cached_k=dev[0], cached_v=dev[1],
                                         depth_valid=Lv or None, moda_group_num=G)
    check_attention(c, q, o, lse, T, G, H, new or [T] * B, scale, plain, depth, L, Lv)


def test_attention_over_a_long_split_cache(gpu_device):
    torch.manual_seed(6)
    past = [20000, 3, 9999]
    for dtype, D in ((BF16, 128), (FP16, 64), (FP32, 64)):
        c = Cache(gpu_device, dtype, 3, 1, D, D, 64, past, [1] * 3)
        q = torch.randn(3, 4, 1, D).to(dtype).to(gpu_device)
        o, lse = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, moda_group_num=4)
        check_attention(c, q, o, lse, 1, 4, 1, [1] * 3, D ** -0.5, False, what=str(dtype))


def test_attention_with_large_logits_and_another_scale(gpu_device):
    """Rows whose weight sits on one key far from the others, early and late: the running maximum jumps."""
    torch.manual_seed(7)
    for dtype in (BF16, FP32):
        c = Cache(gpu_device, dtype, 2, 2, 64, 64, 16, [400, 77], [1, 1])
        q = (30 * torch.randn(2, 4, 2, 64)).to(dtype).to(gpu_device)
        o, lse = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, moda_group_num=4, scale=0.7)
        check_attention(c, q, o, lse, 1, 4, 2, [1, 1], 0.7, False, what=str(dtype))


def test_pages_that_are_not_there(gpu_device):
    """Table entries outside the cache: their tokens are not seen; no page and no slot at all: zero and -inf."""
    torch.manual_seed(8)
    for dtype in (BF16, FP32):
        c = Cache(gpu_device, dtype, 3, 1, 64, 64, 16, [90, 40, 20], [1, 1, 1])
        c.table[0, 2], c.table[0, 4], c.table[1, :], c.table[2, 0] = -7, 2 ** 31 - 1, 10 ** 6, c.k.shape[0]
        q = torch.randn(3, 2, 1, 64).to(dtype).to(gpu_device)
        o, lse = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table.to(gpu_device), c.past_dev, moda_group_num=2)
        keep = [list(range(0, 32)) + list(range(48, 64)) + list(range(80, 91)), [], list(range(16, 21))]
        for b in range(3):
            x, l, e, m = reference_attention(q[b, :, 0].double().cpu(), c.K[b][keep[b], 0].double(), c.V[b][keep[b], 0].double(), 0.125)
            close(o[b, :, 0], x, U[dtype] * x.abs() + (U[dtype] + 2 * e[:, None] + 2.0 ** -16) * m, "o")
            close(lse[b, :, 0], l, e + 2.0 ** -16 + 2.0 ** -22 * l.abs().clamp(max=1e3), "lse")


def test_counts_out_of_range_are_bounded(gpu_device):
    """past below zero counts as zero, past beyond the table as its end, new_lens as 0 .. T."""
    torch.manual_seed(9)
    c = Cache(gpu_device, BF16, 3, 2, 64, 64, 16, [47, 47, 47], [1, 1, 1], spare=0)
    table = c.table_dev[:, :3].contiguous()
    q = torch.randn(3, 1, 2, 64).to(BF16).to(gpu_device)

    def run(past, new=None):
        p = torch.tensor(past, dtype=torch.int32, device=gpu_device)
        n = None if new is None else torch.tensor(new, dtype=torch.int32, device=gpu_device)
        return moda_amd.paged_moda_fwd(q, c.k, c.v, table, p, new_lens=n)

    o, lse = run([-5, 2 ** 31 - 1, 48])
    want, wl = run([0, 47, 47])
    assert torch.equal(o, want) and torch.equal(lse, wl)
    o, lse = run([47] * 3, [9, -3, 1])
    want, wl = run([47] * 3)
    assert torch.equal(o[[0, 2]], want[[0, 2]]) and (o[1] == 0).all() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_values_a_row_does_not_see_may_be_anything(dtype, gpu_device):
    """Non-finite keys and values of later drafted tokens and of other tokens' depth slots reach only the rows that see them."""
    torch.manual_seed(10)
    H, G, D, T, L = 2, 4, 64, 4, 6
    for bad in (math.nan, math.inf):
        c = Cache(gpu_device, dtype, 2, H, D, D, 16, [29, 64], [T, T])
        for b in range(2):
            c.K[b][-1, 0, 3], c.V[b][-2, 1, 5], c.V[b][-1, 1, 9] = bad, bad, -bad
        cc = Cache(gpu_device, dtype, 2, H, D, D, 16, [29, 64], [T, T])
        for b in range(2):
            for j in range(len(c.K[b])):
                cc.k[c.table[b, j // 16], j % 16], cc.v[c.table[b, j // 16], j % 16] = c.K[b][j].to(gpu_device), c.V[b][j].to(gpu_device)
        kd, vd = torch.randn(2, T * L, H, D).to(dtype), torch.randn(2, T * L, H, D).to(dtype)
        vd[:, 2 * L + 1, 0, 7], kd[:, 1 * L + 2, 1, 0] = bad, math.nan
        q = torch.randn(2, T * G, H, D).to(dtype).to(gpu_device)
        o, lse = moda_amd.paged_moda_fwd(q, cc.k, cc.v, c.table_dev, c.past_dev, cached_k=kd.to(gpu_device), cached_v=vd.to(gpu_device),
                                         moda_group_num=G)
        scale = D ** -0.5
        for b in range(2):
            for t in range(T):
                for h in range(H):
                    n = c.past[b] + t + 1
                    keys = torch.cat([c.K[b][:n, h].double(), kd[b, t * L:t * L + L, h].double()])
                    values = torch.cat([c.V[b][:n, h].double(), vd[b, t * L:t * L + L, h].double()])
                    clean = keys.isfinite().all() & values.isfinite().all()
                    rows = o[b, t * G:t * G + G, h]
                    if clean:
                        x, l, e, m = reference_attention(q[b, t * G:t * G + G, h].double().cpu(), keys, values, scale)
                        close(rows, x, U[dtype] * x.abs() + (U[dtype] + 2 * e[:, None] + 2.0 ** -16) * m + TINY[dtype], f"{b} {t} {h}")
                    elif keys.isfinite().all():  # exactly the elements that meet a non-finite value are not finite
                        assert torch.equal(rows.isfinite().all(0).cpu(), values.isfinite().all(0)), (b, t, h)


# ------------------------------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------------------------------

APPEND = [
    # dtype, H, Hq, G, D, Dv, page, T, L, past, new, rotated elements, interleaved, layout
    (BF16, 4, 4, 4, 128, 128, 16, 1, 24, [100], None, 128, False, "tokens"),
    (FP16, 2, 2, 8, 64, 64, 16, 1, 5, [0, 15, 16, 31, 700], None, 64, True, "heads"),
    (BF16, 3, 6, 1, 80, 96, 32, 3, 0, [5, 30, 64], [3, 0, 2], 48, False, "tokens"),
    (FP32, 1, 1, 4, 64, 64, 1, 5, 2, [0, 9], None, 64, False, "tokens"),
    (BF16, 2, 2, 2, 64, 64, 16, 40, 0, [7, 0], [33, 40], 0, False, "heads"),
    (FP16, 2, 4, 1, 64, 32, 64, 70, 0, [0, 100], None, 20, True, "tokens"),
    (FP32, 2, 3, 3, 12, 8, 8, 2, 1, [3, 21], [1, 2], 6, False, "heads"),
    (BF16, 1, 1, 1, 256, 256, 128, 1, 0, [1000000 - 2], None, 256, True, "tokens"),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["padded", "packed"])
def test_append(case, packed, gpu_device):
    dtype, H, Hq, G, D, Dv, P, T, L, past, new, R, inter, layout = case
    torch.manual_seed(12)
    B = len(past)
    new = new or [T] * B
    far = past[0] > 100000
    need = [-(-(p + n) // P) for p, n in zip(past, new)]
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
    n_pages = (4 if far else sum(need)) + 2
    order = torch.randperm(n_pages).int().tolist()
    for b in range(B):
        for i in range(past[b] // P if far else 0, need[b]):
            table[b, i] = order.pop()
    shape = (n_pages, P, H) if layout == "tokens" else (n_pages, H, P)
    ck, cv = (torch.randn(*shape, d).to(dtype).to(gpu_device) for d in (D, Dv))
    if layout == "heads":
        ck, cv = ck.transpose(1, 2), cv.transpose(1, 2)
    if packed:
        total = sum(new) + 3  # three rows behind the last sequence
        at = [sum(new[:b]) for b in range(B)]
        rows = [[(0, at[b] + i) for i in range(new[b])] for b in range(B)]
        tb, tt = 1, total
        counts = {"cu_seqlens": torch.tensor([0] + new).cumsum(0).int().to(gpu_device)}
    else:
        rows = [[(b, i) for i in range(new[b])] for b in range(B)]
        tb, tt = B, T
        counts = {"new_lens": torch.tensor(new, dtype=torch.int32, device=gpu_device)}
    k, v = torch.randn(tb, tt, H, D).to(dtype).to(gpu_device), torch.randn(tb, tt, H, Dv).to(dtype).to(gpu_device)
    q = torch.randn(tb, tt * G, Hq, D).to(dtype).to(gpu_device) if R else None
    rot = moda_amd.Rotary(R, interleaved=inter, scaling="linear", factor=2.0) if R else None
    depth, slot = {}, L // 2
    if L:
        depth = {"cached_k": torch.randn(tb, tt * L, H, D).to(dtype).to(gpu_device), "cached_v": torch.randn(tb, tt * L, H, Dv).to(dtype).to(gpu_device)}
    before = {n: x.cpu().clone() for n, x in dict(depth, ck=ck, cv=cv, k=k, v=v).items()}
    version = ck._version
    q1 = moda_amd.paged_append(k, v, ck, cv, table.to(gpu_device), torch.tensor(past, dtype=torch.int32, device=gpu_device), q=q, rotary=rot,
                               moda_group_num=G, depth_slot=slot, **counts, **depth)
    assert ck._version > version
    # what every row of the batch holds, by its position (rows of no token: padded ones count on, others stay)
    pos = torch.zeros(tb, tt, dtype=torch.long)
    known = torch.zeros(tb, tt, dtype=torch.bool)
    if packed:
        for b in range(B):
            for i, (x, y) in enumerate(rows[b]):
                pos[x, y], known[x, y] = past[b] + i, True
    else:
        pos, known = torch.tensor(past)[:, None] + torch.arange(tt), torch.ones(tb, tt, dtype=torch.bool)
    want_k, tol_k = before["k"].double(), torch.zeros(tb, tt, H, D, dtype=torch.float64)
    if R:
        y, m = rotation64(k, pos, rot)
        want_k, tol_k = y, U[dtype] * y.abs() * (m > 0) + m * 2.0 ** -21 + TINY[dtype] * (m > 0)
        yq, mq = rotation64(q, pos.repeat_interleave(G, 1), rot)
        seen = known.repeat_interleave(G, 1)[..., None, None]
        close(q1, torch.where(seen, yq, q.double().cpu()), torch.where(seen, U[dtype] * yq.abs() * (mq > 0) + mq * 2.0 ** -21 + TINY[dtype] * (mq > 0),
                                                                         torch.zeros(())), "q")
    else:
        assert q1 is None
    ek, ev, tk = before["ck"].double(), before["cv"].double(), torch.zeros(ck.shape, dtype=torch.float64)
    dk, dv, td = (before[n].double() if L else None for n in ("cached_k", "cached_v", "cached_k"))
    td = torch.zeros_like(td) if L else None
    for b in range(B):
        for i, (x, y) in enumerate(rows[b]):
            p = past[b] + i
            at = (int(table[b, p // P]), p % P)
            ek[at], ev[at], tk[at] = want_k[x, y], before["v"][x, y].double(), tol_k[x, y]
            if L:
                r = y * L + slot
                dk[x, r], dv[x, r], td[x, r] = want_k[x, y], before["v"][x, y].double(), tol_k[x, y]
    close(ck, ek, tk, "cache_k")
    close(cv, ev, torch.zeros_like(ev), "cache_v")
    if L:
        close(depth["cached_k"], dk, td, "depth k")
        close(depth["cached_v"], dv, torch.zeros_like(dv), "depth v")


def test_append_takes_offsets_as_they_are(gpu_device):
    """Rows before the first packed sequence, and an offset below the one before it: nowhere, and nothing out of place."""
    torch.manual_seed(19)
    ck, cv = torch.zeros(3, 16, 1, 64, device=gpu_device), torch.zeros(3, 16, 1, 64, device=gpu_device)
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32, device=gpu_device)
    past = torch.zeros(3, dtype=torch.int32, device=gpu_device)
    k, v, q = (torch.randn(1, 9, 1, 64, device=gpu_device) for _ in range(3))
    rot = moda_amd.Rotary(64)
    cu = torch.tensor([2, 4, 4, 7], dtype=torch.int32, device=gpu_device)
    q1 = moda_amd.paged_append(k, v, ck, cv, table, past, cu_seqlens=cu, q=q, rotary=rot)
    want = torch.zeros_like(cv)
    want[0, :2], want[2, :3] = v[0, 2:4], v[0, 4:7]
    assert torch.equal(cv, want)
    assert torch.equal(q1[:, :2], q[:, :2]) and torch.equal(q1[:, 7:], q[:, 7:])
    for offsets in ([0, 5, 2, 9], [9, 0, -4, 2 ** 31 - 1], [-7, -5, -3, -1]):
        cv.zero_()
        moda_amd.paged_append(k, v, ck, cv, table, past, cu_seqlens=torch.tensor(offsets, dtype=torch.int32, device=gpu_device))
        rows = {tuple(r) for r in v[0, :, 0].tolist()} | {(0.0,) * 64}
        assert {tuple(r) for r in cv.view(-1, 64).tolist()} <= rows


def test_append_drops_what_has_no_place(gpu_device):
    torch.manual_seed(13)
    ck, cv = torch.zeros(4, 16, 1, 64, dtype=BF16, device=gpu_device), torch.zeros(4, 16, 1, 64, dtype=BF16, device=gpu_device)
    table = torch.tensor([[2, -1, 1], [4, 3, 2 ** 31 - 1], [-2 ** 31, 0, 9]], dtype=torch.int32, device=gpu_device)
    past = torch.tensor([10, 10, -4], dtype=torch.int32, device=gpu_device)
    k, v = torch.randn(3, 50, 1, 64, device=gpu_device).to(BF16), torch.randn(3, 50, 1, 64, device=gpu_device).to(BF16)
    moda_amd.paged_append(k, v, ck, cv, table, past)
    for x, c in ((k, ck), (v, cv)):
        want = torch.zeros_like(c)
        want[2, 10:] = x[0, :6]
        want[1] = x[0, 22:38]      # positions 32 .. 47; what is past the table's 48 positions is dropped
        want[3] = x[1, 6:22]
        want[0] = x[2, 16:32]      # a count below zero counts as zero
        assert torch.equal(c, want)


# ------------------------------------------------------------------------------------------------------------------
# together, and where a call runs
# ------------------------------------------------------------------------------------------------------------------


def test_steps_of_a_layer_agree_with_the_whole_sequence(gpu_device):
    """A sequence written and read token by token -- rotation, append, attention, depth slots -- is the causal operator's."""
    torch.manual_seed(14)
    B, T, H, G, D, L = 2, 45, 2, 4, 64, 5
    rot = moda_amd.Rotary(64, base=500.0)
    q, k, v = (torch.randn(B, T * n, H, D, device=gpu_device).to(BF16) for n in (G, 1, 1))
    kd, vd = (torch.randn(B, T * L, H, D, device=gpu_device).to(BF16) for _ in range(2))
    qr, kr = moda_amd.apply_rotary(q, k, rot, moda_group_num=G)
    want = moda_amd.parallel_moda(qr, kr, v, cached_k=kd, cached_v=vd, moda_group_num=G, is_causal=True, depth_valid=3)
    cache = moda_amd.PagedKVCache(1, 8, 16, H, D, BF16, gpu_device, batch=B, max_tokens=64)
    for b in range(B):
        cache.reserve(b, T)
    got, at = [], 0
    with torch.no_grad():
        for n in (20, 1, 1, 3, 1, 5, 1, 13):
            rows, slots = slice(at * G, (at + n) * G), slice(at * L, (at + n) * L)
            q1 = cache.append(0, k[:, at:at + n], v[:, at:at + n], q=q[:, rows], rotary=rot, moda_group_num=G)
            assert torch.equal(q1, qr[:, rows])
            got.append(cache.attend(0, q1, cached_k=kd[:, slots], cached_v=vd[:, slots], depth_valid=3, moda_group_num=G))
            cache.advance(n)
            at += n
    got = torch.cat(got, 1)
    # both round their probabilities and their results to 16 bits: |o| and sum p |v| are at most the largest value
    tol = 4 * U[BF16] * torch.full(want.shape, float(v.abs().max().clamp(min=vd.abs().max())))
    close(got, want.detach(), tol, "o")
    err = (got.double() - want.double()).norm() / want.double().norm()
    assert err < 2 * U[BF16], float(err)
    assert cache.past.tolist() == [T, T]


def _step(c, q, k, v, rot, depth):
    q1 = moda_amd.paged_append(k, v, c.k, c.v, c.table_dev, c.past_dev, q=q, rotary=rot, moda_group_num=4, cached_k=depth[0], cached_v=depth[1],
                               depth_slot=2)
    return moda_amd.paged_moda_fwd(q1, c.k, c.v, c.table_dev, c.past_dev, cached_k=depth[0], cached_v=depth[1], depth_valid=3, moda_group_num=4)


def test_captured_step_replays_as_lengths_grow(gpu_device):
    torch.manual_seed(15)
    dev = gpu_device
    c = Cache(dev, BF16, 2, 2, 64, 64, 16, [5, 600], [40, 40])
    rot = moda_amd.Rotary(64)
    q, k, v = (torch.randn(2, n, 2, 64, device=dev).to(BF16) for n in (4, 1, 1))
    depth = [torch.randn(2, 4, 2, 64, device=dev).to(BF16) for _ in range(2)]
    _step(c, q, k, v, rot, depth)
    first = c.past_dev.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        _step(c, q, k, v, rot, depth)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o, lse = _step(c, q, k, v, rot, depth)
        c.past_dev.add_(1)
    c.past_dev.copy_(first)
    for i in range(12):
        for x in (q, k, v):
            x.normal_()
        saved = c.past_dev.clone()
        graph.replay()
        got = o.clone(), lse.clone()
        assert c.past_dev.tolist() == (saved + 1).tolist()
        c.past_dev.copy_(saved)
        want = _step(c, q, k, v, rot, depth)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        c.past_dev.add_(1 if i % 2 else 3)


def test_two_captured_graphs_and_two_streams(gpu_device):
    """Calls at the same time have their own work areas: two graphs replayed on two streams, with eager calls between."""
    torch.manual_seed(16)
    dev = gpu_device
    calls = []
    for past in ([3000, 41], [17, 2200, 900]):
        c = Cache(dev, BF16, len(past), 2, 128, 128, 16, past, [1] * len(past))
        q = torch.randn(len(past), 4, 2, 128, device=dev).to(BF16)
        calls.append(lambda c=c, q=q: moda_amd.paged_moda(q, c.k, c.v, c.table_dev, c.past_dev, moda_group_num=4))
    want = [f() for f in calls]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for f in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f())
    for _ in range(6):
        for s, g, o in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                o.fill_(7)
                g.replay()
        eager = [f() for f in calls]
        torch.cuda.synchronize()
        for a, b, w in zip(outs, eager, want):
            assert torch.equal(a, w) and torch.equal(b, w)


def test_captured_backward_of_a_rotation(gpu_device):
    rot = moda_amd.Rotary(64)
    x, w = torch.randn(1, 30, 2, 64, device=gpu_device), torch.randn(1, 30, 2, 64, device=gpu_device)

    def run():
        leaf = x.detach().requires_grad_()
        y = moda_amd.apply_rotary(leaf, None, rot)[0]
        return y.detach(), torch.autograd.grad(y, leaf, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, d = run()
    for _ in range(5):
        x.normal_(), w.normal_()
        g.replay()
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(d, want[1])


def test_results_do_not_change_from_run_to_run(gpu_device):
    torch.manual_seed(17)
    c = Cache(gpu_device, BF16, 4, 2, 128, 128, 16, [5000, 1, 333, 2047], [1] * 4)
    q = torch.randn(4, 4, 2, 128, device=gpu_device).to(BF16)
    first = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, moda_group_num=4)
    for _ in range(10):
        again = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, moda_group_num=4)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_cache_beyond_four_gibibytes(gpu_device):
    """Offsets that pass 32 bits, in bytes and in elements: pages at both ends of a cache of 2^32 elements."""
    H, D, P = 8, 128, 64
    n = 2 ** 32 // (P * H * D) + 3
    ck = torch.zeros(n, P, H, D, dtype=BF16, device=gpu_device)
    cv = torch.zeros(n, P, H, D, dtype=BF16, device=gpu_device)
    table = torch.tensor([[n - 1, 0, n - 2], [1, n - 3, 2]], dtype=torch.int32)
    past = torch.tensor([0, 0], dtype=torch.int32, device=gpu_device)
    torch.manual_seed(18)
    k, v = torch.randn(2, 150, H, D).to(BF16), torch.randn(2, 150, H, D).to(BF16)
    moda_amd.paged_append(k.to(gpu_device), v.to(gpu_device), ck, cv, table.to(gpu_device), past)
    for b in range(2):
        for j in (0, 63, 64, 127, 128, 149):
            assert torch.equal(ck[table[b, j // P], j % P].cpu(), k[b, j]) and torch.equal(cv[table[b, j // P], j % P].cpu(), v[b, j])
    q = torch.randn(2, 2, H, D).to(BF16).to(gpu_device)
    past.fill_(149)
    o, lse = moda_amd.paged_moda_fwd(q, ck, cv, table.to(gpu_device), past, moda_group_num=2)

    class C:
        K, V, past = [k[0], k[1]], [v[0], v[1]], [149, 149]
    check_attention(C, q, o, lse, 1, 2, H, [1, 1], D ** -0.5, False)


# ------------------------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------------------------


def test_refusals(gpu_device):
    dev = gpu_device
    rot = moda_amd.Rotary(64)
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    q, k = z(1, 8, 2, 64), z(1, 4, 2, 64)
    for kw, exc in ((dict(moda_group_num=3), AssertionError), (dict(moda_group_num=0), AssertionError),
                    (dict(positions=torch.zeros(4)), AssertionError), (dict(positions=torch.zeros(4, dtype=torch.int64)), AssertionError),
                    (dict(positions=torch.zeros(3, dtype=torch.int64, device=dev)), AssertionError),
                    (dict(positions=torch.zeros(4, device=dev)), AssertionError), (dict(rotary=moda_amd.Rotary(66)), AssertionError),
                    (dict(k=z(1, 4, 2, 64, dtype=FP16)), TypeError), (dict(k=z(1, 4, 2, 32)), AssertionError), (dict(k=z(2, 4, 2, 64)), AssertionError),
                    (dict(q=z(8, 2, 64)), AssertionError), (dict(q=z(1, 8, 2, 64).double(), k=None), TypeError)):
        args = dict(q=q, k=k, rotary=rot, moda_group_num=2)
        args.update(kw)
        with pytest.raises(exc):
            moda_amd.apply_rotary(**args)

    ck, table, past = z(4, 16, 2, 64), z(1, 3, dtype=torch.int32), z(1, dtype=torch.int32)
    good = dict(q=z(1, 4, 2, 64), cache_k=ck, cache_v=ck.clone(), page_table=table, past=past, moda_group_num=4)
    moda_amd.paged_moda(**good)
    bad = [dict(q=z(1, 4, 3, 64)), dict(q=z(1, 4, 2, 32)), dict(q=z(4, 2, 64)), dict(q=z(2, 4, 2, 64)), dict(moda_group_num=3), dict(moda_group_num=0),
           dict(q=z(1, 4, 2, 64, dtype=FP16)), dict(cache_v=z(4, 16, 2, 64, dtype=FP16)), dict(cache_v=z(4, 8, 2, 64)), dict(cache_k=z(4, 12, 2, 64), cache_v=z(4, 12, 2, 64)),
           dict(cache_k=z(0, 16, 2, 64), cache_v=z(0, 16, 2, 64)), dict(cache_k=z(4, 16, 2, 68)[..., :64]), dict(cache_k=z(4, 16, 64, 2).transpose(2, 3)),
           dict(page_table=table.long()), dict(page_table=table.cpu()), dict(page_table=z(2, 3, dtype=torch.int32)), dict(page_table=z(1, 0, dtype=torch.int32)),
           dict(past=past.long()), dict(past=z(2, dtype=torch.int32)), dict(past=past.cpu()), dict(new_lens=z(2, dtype=torch.int32)), dict(new_lens=z(1)),
           dict(cached_k=z(1, 5, 2, 64), cached_v=z(1, 4, 2, 64)), dict(cached_k=z(1, 5, 2, 64), cached_v=z(1, 5, 2, 64), depth_valid=6),
           dict(cached_k=z(1, 5, 2, 64), cached_v=z(1, 5, 2, 64), depth_valid=0), dict(cached_k=z(1, 5, 1, 64), cached_v=z(1, 5, 1, 64)),
           dict(q=z(1, 4, 2, 64).requires_grad_()), dict(q=z(2, 6, 2, 64), page_table=z(2, 3, dtype=torch.int32), past=z(2, dtype=torch.int32), moda_group_num=2,
                                                         cached_k=z(2, 5, 2, 64), cached_v=z(2, 5, 2, 64))]
    for kw in bad:
        with pytest.raises((AssertionError, TypeError)):
            moda_amd.paged_moda(**{**good, **kw})
    for dim in (12, 264):
        with pytest.raises((RuntimeError, AssertionError)):
            moda_amd.paged_moda(z(1, 4, 2, dim), z(4, 16, 2, dim), z(4, 16, 2, dim), table, past, moda_group_num=4)
    with torch.no_grad():  # nothing to differentiate: fine
        moda_amd.paged_moda(**{**good, "q": z(1, 4, 2, 64).requires_grad_()})
    with pytest.raises(AssertionError):
        moda_amd.paged_attn(z(1, 1, 5, 64), ck, ck, table, past)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda q: moda_amd.paged_moda(q, ck, ck, table, past, moda_group_num=4), (z(1, 4, 2, 64),), check_trace=False)

    cv = z(4, 16, 2, 64)
    good = dict(k=z(1, 3, 2, 64), v=z(1, 3, 2, 64), cache_k=ck, cache_v=cv, page_table=table, past=past)
    moda_amd.paged_append(**good)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    moda_amd.paged_append(**good, cu_seqlens=cu)
    for kw in (dict(k=z(1, 3, 1, 64)), dict(v=z(1, 2, 2, 64)), dict(k=z(1, 3, 2, 32)), dict(k=z(3, 2, 64)), dict(k=z(1, 3, 2, 64, dtype=FP16)),
               dict(k=z(1, 3, 2, 64).requires_grad_()), dict(cache_k=z(4, 16, 2, 64).requires_grad_()), dict(q=z(1, 3, 2, 64)), dict(q=z(1, 5, 2, 64), rotary=rot, moda_group_num=2),
               dict(rotary=moda_amd.Rotary(66)), dict(cu_seqlens=cu, new_lens=past), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu.cpu()),
               dict(cached_k=z(1, 6, 2, 64)), dict(cached_k=z(1, 6, 2, 64), cached_v=z(1, 6, 2, 64), depth_slot=2),
               dict(cached_k=z(1, 7, 2, 64), cached_v=z(1, 7, 2, 64)), dict(cache_k=z(1, 16, 2, 64).expand(4, 16, 2, 64)),
               dict(cached_k=z(1, 6, 2, 128)[..., :64], cached_v=z(1, 6, 2, 64))):
        with pytest.raises((AssertionError, TypeError)):
            moda_amd.paged_append(**{**good, **kw})
    assert moda_amd.paged_append(z(1, 0, 2, 64), z(1, 0, 2, 64), ck, cv, table, past) is None
    assert moda_amd.paged_append(z(1, 0, 2, 64), z(1, 0, 2, 64), ck, cv, table, past, cached_k=z(1, 0, 2, 64), cached_v=z(1, 0, 2, 64)) is None
    assert moda_amd.paged_moda(z(1, 0, 2, 64), ck, cv, table, past).shape == (1, 0, 2, 64)
    assert moda_amd.paged_moda(z(0, 4, 2, 64), ck, cv, z(0, 3, dtype=torch.int32), z(0, dtype=torch.int32), moda_group_num=4).shape == (0, 4, 2, 64)
