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

from test_paged_gpu import ATTEND, Cache

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


@pytest.mark.parametrize("gap", [12, 18, 22, 26, 33, 40])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_small_probabilities_count_in_the_sums_and_in_the_result(dtype, gap, gpu_device):
    """A first key `gap` bits ahead of 4000 others and without a value, as of a model that parks its attention there: the result is made
    of the others alone.  So many sequences (of the same pages) that a wave has all keys of one in its run; and the same in many runs."""
    g = torch.Generator().manual_seed(32)
    H, D, Dv, n = 8, 8, 8, 4001
    keys, values = torch.zeros(1, n, H, D, dtype=dtype), torch.zeros(1, n, H, Dv, dtype=dtype)
    keys[:, 1:, :, 0] = (-(gap + torch.rand(1, n - 1, H, generator=g)) * math.log(2)).to(dtype)
    values[:, 1:] = ((1 + torch.rand(1, n - 1, H, Dv, generator=g)) * 2.0 ** min(gap - 12, 14)).to(dtype)
    p = torch.exp(keys[..., :1].double())
    want, lse = (p * values.double()).sum(1) / p.sum(1), torch.log2(p.sum(1))[..., 0]
    # logits of at most gap + 1; off by e and, against what they are taken, by 2^-24 of their size and 15; the sums: 32 keys of a tile
    # in three pieces, the tiles and their changes of scale, parts
    e = 2.0 ** -23 * (gap + 1.1) + 2.0 ** -24 * (gap + 17)
    depth = (96 + 2 * 126 + 16) * 2.0 ** -24
    tol = U[dtype] * want.abs() + (2 * math.log(2) * e + 3 * 2.0 ** -23 + 2 * depth) * want.abs() + n * 2.0 ** (15 - 64) + TINY[dtype]
    ck, cv, table, past = pages_of(keys, values, gpu_device)
    for B in (384, 1):
        q = torch.zeros(B, 1, H, D, dtype=dtype)
        q[..., 0] = 1
        o, l = moda_amd.paged_moda_fwd(q.to(gpu_device), ck, cv, table.expand(B, -1), past.expand(B).contiguous(), scale=1.0)
        within(o[:, 0].double().cpu(), want.expand(B, -1, -1), tol.expand(B, -1, -1), f"o of {B}")
        within(l[:, 0].double().cpu(), lse.expand(B, -1), torch.full((B, H), math.log(2) * e + depth + 2.0 ** -21), f"lse of {B}")


def test_fp16_logits_too_large_to_count_in_ones(gpu_device):
    """Logits of 2^24 and more, where numbers are further apart than one: the largest probability stays what the type can hold."""
    for size in (2.0 ** 11, 2.0 ** 12, 2.0 ** 12 + 4, 30000.0, 60000.0):
        keys, values = torch.full((1, 40, 1, 8), size / 2, dtype=FP16), torch.zeros(1, 40, 1, 8, dtype=FP16)
        keys[0, 17], values[0, 17] = size, 3.0
        q = torch.full((1, 1, 1, 8), size, dtype=FP16)
        o, lse = moda_amd.paged_moda_fwd(q.to(gpu_device), *pages_of(keys, values, gpu_device), scale=1.0)
        assert (o == 3).all(), (size, o)
        exact = 8 * size * size * math.log2(math.e)
        assert abs(float(lse) - exact) <= exact * 12 * 2.0 ** -24, size


def attention64(q, keys, values, scale):
    """q [rows, D], keys [n, D], values [n, Dv] in 64 bits -> o, lse (base 2), and what they may be off by before o is rounded: logits of D
    products and a scale (e); a probability of the last unit of its exponential; sums of n terms in any order."""
    s = q @ keys.T * (scale / math.log(2))
    lse = torch.logsumexp(s * math.log(2), -1) / math.log(2)
    p = torch.exp2(s - lse[:, None])
    e = (q.abs() @ keys.abs().T).amax(-1) * (scale / math.log(2)) * (q.shape[1] + 4) * 2.0 ** -24
    n = keys.shape[0]
    finite = values.masked_fill(~values.isfinite(), 0)
    tol = (2 * math.log(2) * e[:, None] + (2 * n + 100) * 2.0 ** -24) * (p @ finite.abs())
    return p @ values, lse, tol, e + (n + 20) * 2.0 ** -24 + 2.0 ** -22 * lse.abs().clamp(min=1)


def same(got, want, tol, what):
    """Equal where the reference is not finite (NaN with NaN, infinities by their sign), else within tol."""
    got, want = got.double().cpu(), want.double()
    odd = ~want.isfinite()
    assert torch.equal(got[odd].isnan(), want[odd].isnan()) and bool((got[odd] == want[odd])[~want[odd].isnan()].all()), \
        f"{what}: {got[odd][:8].tolist()} for {want[odd][:8].tolist()}"
    within(got.masked_fill(odd, 0), want.masked_fill(odd, 0), tol.masked_fill(odd, 1), what)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("T,G,D", [(1, 4, 64), (1, 1, 128), (1, 8, 256), (1, 40, 64), (4, 4, 64), (3, 8, 64), (5, 8, 64), (3, 8, 128), (9, 8, 128), (5, 8, 256),
                                   (5, 3, 80)], ids=str)
def test_values_and_keys_that_are_not_finite(dtype, T, G, D, gpu_device):
    """Infinities and NaN in values, early, in the middle and at the end, seen by all rows, by some, and by one token's alone; NaN in a
    key.  What a row sees of them is in its result -- inf as inf, inf and -inf as NaN -- and nothing else is; rows of 16 and fewer, of a tile of
    32 and of several tiles."""
    g = torch.Generator().manual_seed(33)
    B, H, L, Lv, n = 3, 2, 6, 5, 231
    keys, values = torch.randn(B, n, H, D, generator=g).to(dtype), torch.randn(B, n, H, D, generator=g).to(dtype)
    kd, vd = torch.randn(B, T * L, H, D, generator=g).to(dtype), torch.randn(B, T * L, H, D, generator=g).to(dtype)
    q = torch.randn(B, T * G, H, D, generator=g).to(dtype)
    inf, nan = math.inf, math.nan
    values[0, 3, 0, 1], values[0, 100, 0, 2], values[0, 50, 0, 4], values[0, n - 1, 0, 5] = inf, -inf, nan, inf
    values[0, 3, 0, 3], values[0, 180, 0, 3] = inf, -inf
    values[1, n - 1, 1, D - 1], values[1, n - 2, 1, D - 2], vd[1, (T - 1) * L + 2, 0, 6], vd[1, 0, 1, 7] = -inf, inf, -inf, nan
    vd[:, Lv::L], kd[:, Lv::L] = nan, nan  # slots that are not valid
    keys[2, n - 1, 0, 0], kd[2, 1, 1, 2] = nan, nan
    past = torch.full((B,), n - T, dtype=torch.int32, device=gpu_device)
    ck, cv, table, _ = pages_of(keys, values, gpu_device)
    o, lse = moda_amd.paged_moda_fwd(q.to(gpu_device), ck, cv, table, past, cached_k=kd.to(gpu_device), cached_v=vd.to(gpu_device), depth_valid=Lv,
                                     moda_group_num=G)
    for b in range(B):
        for t in range(T):
            for h in range(H):
                seen = n - T + t + 1
                slots = slice(t * L, t * L + Lv)
                k, v = (torch.cat([x[b, :seen, h], y[b, slots, h]]).double() for x, y in ((keys, kd), (values, vd)))
                rows = (b, slice(t * G, t * G + G), h)
                if k.isnan().any():
                    assert o[rows].isnan().all() and lse[rows].isnan().all(), (b, t, h)
                    continue
                x, l, tol, tl = attention64(q[rows].double(), k, v, D ** -0.5)
                same(o[rows], x, tol + U[dtype] * x.abs() + TINY[dtype], f"o {b} {t} {h}")
                same(lse[rows], l, tl, f"lse {b} {t} {h}")


def rounded_attention64(q, keys, values, scale, dtype, tiles):
    """q [rows, D] in 64 bits -> o, lse and how far a call in `dtype` may be from them where its probabilities meet the values with all their
    bits.  `tiles`: of 32 keys in the whole call, of which a wave of a thousand or more has an equal run, in order: each key is added in
    at most three pieces (96 additions a tile), the tiles bring sums to a new scale, and the runs of a row are joined."""
    s = q @ keys.T * (scale / math.log(2))
    lse = torch.logsumexp(s * math.log(2), -1) / math.log(2)
    p = torch.exp2(s - lse[:, None])
    o, magnitude = p @ values, p @ values.abs()
    e = (q.abs() @ keys.abs().T).amax(-1) * (scale / math.log(2)) * (q.shape[1] + 4) * 2.0 ** -24
    sums = (98 * -(-tiles // 1024) + -(-keys.shape[0] // 32) + 20) * 2.0 ** -24
    return o, lse, U[dtype] * o.abs() + (2 * math.log(2) * e[:, None] + 2 * sums + 2.0 ** -21) * magnitude + TINY[dtype], \
        e + sums + 2.0 ** -21 + 2.0 ** -23 * lse.abs()


def check_rounded(c, q, o, lse, T, G, H, new, scale, plain, depth=None, L=0, Lv=0):
    """`c`: K, V of each sequence and past, on the CPU (test_paged_gpu.Cache)."""
    lengths = [c.past[b] + new[b] if new[b] else 0 for b in range(q.shape[0])]
    tiles = H * -(-T * G // 16) * sum(-(-n // 32) + (T * -(-Lv // 16) + 1) // 2 + 1 for n in lengths)
    for b in range(q.shape[0]):
        for t in range(T):
            for h in range(H):
                at = (b, t, slice(h * G, h * G + G)) if plain else (b, slice(t * G, t * G + G), h)
                if t >= new[b]:
                    assert (o[at] == 0).all() and (lse[at] == -math.inf).all(), (b, t, h)
                    continue
                keys, values = c.K[b][:c.past[b] + t + 1, h].double(), c.V[b][:c.past[b] + t + 1, h].double()
                if depth:
                    r = slice(t * L, t * L + Lv)
                    keys, values = torch.cat([keys, depth[0][b, r, h].double()]), torch.cat([values, depth[1][b, r, h].double()])
                x, l, tol, tl = rounded_attention64(q[at].double().cpu(), keys, values, scale, q.dtype, tiles)
                within(o[at].double().cpu(), x, tol, f"o {b} {t} {h}")
                within(lse[at].double().cpu(), l, tl, f"lse {b} {t} {h}")


@pytest.mark.parametrize("case", ATTEND, ids=str)
@pytest.mark.parametrize("plain", [False, True], ids=["folded", "plain"])
def test_attention_is_at_its_rounding(case, plain, gpu_device):
    """The cases of the test of attention over pages, without an allowance for probabilities in 16 bits."""
    dtype, H, G, D, Dv, P, T, L, Lv, past, new, layout = case
    if plain:
        L = Lv = 0
    torch.manual_seed(51)
    B = len(past)
    new = new or [T] * B
    c = Cache(gpu_device, dtype, B, H, D, Dv, P, past, new, layout)
    q = torch.randn((B, T, H * G, D) if plain else (B, T * G, H, D)).to(dtype).to(gpu_device)
    lens = torch.tensor(new, dtype=torch.int32, device=gpu_device)
    depth = None
    if plain:
        o, lse = moda_amd.paged_attn_fwd(q, c.k, c.v, c.table_dev, c.past_dev, new_lens=lens)
    else:
        if L:
            depth = torch.randn(B, T * L, H, D).to(dtype), torch.randn(B, T * L, H, Dv).to(dtype)
        dev = [x.to(gpu_device) for x in depth] if depth else [None, None]
        o, lse = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, new_lens=lens, cached_k=dev[0], cached_v=dev[1], depth_valid=Lv or None,
                                         moda_group_num=G)
    check_rounded(c, q, o, lse, T, G, H, new, D ** -0.5, plain, depth, L, Lv)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64), (FP32, 64), (BF16, 256)], ids=str)
def test_a_long_split_cache_is_at_its_rounding(dtype, D, gpu_device):
    """What one tile of values too few or in a wrong place would change is more than this allows (tests/test_paged_tolerance_cpu.py)."""
    torch.manual_seed(52)
    past = [20000, 3, 9999]
    c = Cache(gpu_device, dtype, 3, 1, D, D, 64, past, [1] * 3)
    q = torch.randn(3, 4, 1, D).to(dtype).to(gpu_device)
    o, lse = moda_amd.paged_moda_fwd(q, c.k, c.v, c.table_dev, c.past_dev, moda_group_num=4)
    check_rounded(c, q, o, lse, 1, 4, 1, [1] * 3, D ** -0.5, False)
