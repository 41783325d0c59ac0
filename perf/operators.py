"""The operators of generation with a paged key/value cache, and the rotary positions they share with training: what is
measured, as plain torch operations (``own = False``) and as calls of this package's kernels (``own = True``).

  op      rotary  ``apply_rotary`` on q and k (``grad``: with its backward pass)
          append  ``paged_append``: K (rotated) and V of new tokens into their pages and depth slots, q rotated
          attend  ``paged_moda`` (folded query rows, depth slots) or, with ``plain``, ``paged_attn``
  dtype   bf16 | fp16 | fp32
  B, T    sequences, new tokens of each;  ``ragged``: the last sequences have fewer new tokens (``append``: packed with
          offsets, ``attend``: padded)
  H, G    key/value heads, query heads on each;  D: head dim
  lo, hi  tokens of a sequence before the call (spread between the two); for ``rotary`` the first position
  page    tokens per page
  L, n    depth slots per token and how many of them hold data (``append``: n is the slot written)
  rot     elements of a head that are rotated (0: none);  ``pairs``: half | inter;  ``scaling``, ``factor``, ``orig``
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BASE = 10000.0

_PACKED_LENGTHS = [16384] + [8192] * 2 + [4096] * 4 + [2048] * 8


def _case(op, B, T, H, G, D, dtype="bf16", lo=0, hi=None, page=0, L=0, n=0, rot=0, pairs="half", scaling="none", factor=1.0,
          orig=0, grad=False, ragged=False, plain=False, lens=""):
    return {"op": op, "B": B, "T": T, "H": H, "G": G, "D": D, "dtype": dtype, "lo": lo, "hi": lo if hi is None else hi,
            "page": page, "L": L, "n": n, "rot": rot, "pairs": pairs, "scaling": scaling, "factor": factor, "orig": orig,
            "grad": grad, "ragged": ragged, "plain": plain, "lens": lens}


def listed():
    cases = {
        # the query and key of one generated token: a launch and the host time of the call are all of it
        "rotary-token": _case("rotary", 1, 1, 4, 4, 128, lo=5000, rot=128),
        # a layer of the long-context training step, forward and backward
        "rotary-64k-train": _case("rotary", 1, 65536, 4, 4, 128, rot=128, grad=True),
        # fp32 fine-tuning of a smaller model on far positions: half of each head rotated in neighbouring pairs, angles
        # scaled for eight times the length, odd sizes
        "rotary-part-train": _case("rotary", 3, 1021, 6, 1, 64, "fp32", lo=500000, rot=32, pairs="inter", scaling="by_parts",
                                   factor=8.0, orig=65536, grad=True),
        # one new token of one sequence, K and V also into the token's depth slot
        "append-token": _case("append", 1, 1, 4, 4, 128, lo=1000, page=16, L=24, n=5, rot=128),
        # one new token for each of many sequences of different lengths, 64 query heads
        "append-batch": _case("append", 256, 1, 8, 8, 64, "fp16", lo=1, hi=511, page=16, L=64, n=17, rot=64),
        # prompts of different lengths, packed on one token axis
        "append-prompts": _case("append", len(_PACKED_LENGTHS), 16384, 4, 4, 128, page=64, rot=128, ragged=True,
                                lens=",".join(map(str, _PACKED_LENGTHS))),
        # the first tokens of an answer: a short cache
        "attend-token": _case("attend", 1, 1, 4, 4, 128, lo=100, page=16, L=24, n=8),
        # ordinary serving: a batch of sequences of 1 K to 8 K tokens
        "attend-batch": _case("attend", 64, 1, 4, 4, 128, lo=1000, hi=8100, page=16, L=24, n=23),
        # one very long sequence: everything is in the split of its length
        "attend-long": _case("attend", 1, 1, 4, 4, 128, lo=1048575, page=64, L=24, n=12),
        # five drafted tokens (fewer for some sequences) to be verified, eight query heads a key/value head, short and long
        "attend-drafts": _case("attend", 16, 5, 8, 8, 64, "fp16", lo=0, hi=4000, page=32, L=64, n=33, ragged=True),
        # fp32, as gradient checks and small models use it
        "attend-fp32": _case("attend", 2, 1, 4, 1, 64, "fp32", lo=1500, hi=2100, page=16, L=4, n=3),
        # the largest batch, whose cache passes 4 GiB; layers that carry no depth stream
        "attend-wide": _case("attend", 256, 1, 4, 4, 128, lo=12000, hi=24000, page=128, plain=True),
    }
    return [dict(c, name=k) for k, c in cases.items()]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm, odd as often as even."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    top = work(next(c for c in listed() if c["name"] == "attend-wide"))["bytes"]
    while True:
        c = _draw_any(rng)
        # plain forms gather whole tables in 32 bits, and small launches run at a lower rate: leave room for that
        longest = c["B"] * max(_lengths(c)) * c["H"] * c["D"] * _SIZES[c["dtype"]]
        if c["op"] == "rotary" and work(c)["bytes"] <= top / 32 or c["op"] == "append" and longest <= top / 32 or \
                c["op"] == "attend" and longest <= top / 4:
            return c


def _draw_any(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    D = rng.choice([64, 64, 80, 96, 128, 128, 192, 256])
    H, G = rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 2, 3, 4, 8])
    rot = dict(rot=D if rng.random() < 0.6 else 16 * rng.randint(1, D // 16), pairs=rng.choice(["half", "inter"]))
    rot["scaling"] = rng.choice(["none", "none", "linear", "ntk", "by_parts"])
    rot.update(factor=1.0 if rot["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0]), orig=rng.choice([4096, 32768]))
    if op == "rotary":
        return _case(op, _between(rng, 1, 16), _between(rng, 1, 32768), H, G, D, dtype,
                     lo=rng.choice([0, _between(rng, 1, 1000000)]), grad=rng.random() < 0.6, **rot)
    L = rng.choice([0, _between(rng, 2, 64)])
    page, B = rng.choice([16, 32, 64, 128]), _between(rng, 1, 256)
    if op == "append":
        T = rng.choice([1, 1, _between(rng, 2, 4096)])
        past = _between(rng, 1, 2000)
        return _case(op, B, T, H, G, D, dtype, lo=rng.randint(0, past), hi=past, page=page, L=L, n=rng.randrange(L) if L else 0,
                     ragged=T > 1 and L == 0 and rng.random() < 0.5, **(rot if rng.random() < 0.8 else {}))
    hi = _between(rng, 16, 300000)
    T = rng.choice([1, 1, 1, rng.randint(2, 8)])
    plain = rng.random() < 0.3
    L = 0 if plain else L
    return _case(op, B, T, H, G, D, dtype, lo=rng.choice([hi, 0, hi // 4]), hi=hi, page=page, L=L, n=rng.randint(1, L) if L else 0,
                 ragged=T > 1 and rng.random() < 0.5, plain=plain)


# ------------------------------------------------------------------------------------------------------------------
# what a case holds
# ------------------------------------------------------------------------------------------------------------------


def _past(c):
    """Tokens of each sequence before the call, spread between lo and hi."""
    return [c["lo"] + int((c["hi"] - c["lo"]) * ((b * 0.6180339887498949 + 0.999) % 1.0) + 0.5) for b in range(c["B"])]


def _new(c):
    """New tokens of each sequence."""
    if c["lens"]:
        return [int(x) for x in c["lens"].split(",")]
    if not c["ragged"]:
        return [c["T"]] * c["B"]
    return [c["T"] - (b * 7 + 3) % (c["T"] + 1) for b in range(c["B"])]


def _lengths(c):
    return [p + n for p, n in zip(_past(c), _new(c))]


def _rates(c):
    """Turns per position of each rotated pair, in 64 bits, and the factor on the rotated elements."""
    R, s = c["rot"], c["factor"]
    base = _BASE * s ** (R / (R - 2)) if c["scaling"] == "ntk" else _BASE
    f = torch.tensor([base ** (-2 * i / R) / (2 * math.pi) for i in range(R // 2)], dtype=torch.float64)
    if c["scaling"] == "linear":
        f = f / s
    if c["scaling"] == "by_parts":
        keep = ((f * c["orig"] - 1) / 31).clamp(0, 1)
        return f / s * (1 - keep) + f * keep, 0.1 * math.log(s) + 1
    return f, 1.0


def work(c):
    es, H, G, D = _SIZES[c["dtype"]], c["H"], c["G"], c["D"]
    if c["op"] == "rotary":
        tokens, heads, passes = c["B"] * c["T"], H * (G + 1), 2 if c["grad"] else 1
        return {"bytes": passes * tokens * (2 * heads * D * es + 8), "flops": passes * tokens * heads * c["rot"] * 3}
    new, rows = sum(_new(c)), H * D * es
    if c["op"] == "append":
        q = 2 * G * rows if c["rot"] else 0
        return {"bytes": new * (2 * rows * (2 if c["L"] == 0 else 3) + q), "flops": new * H * (G + 1) * c["rot"] * 3}
    seen = sum(max(0, p * n + n * (n + 1) // 2) for p, n in zip(_past(c), _new(c)))  # (token, key) pairs
    keys = sum(l for l, n in zip(_lengths(c), _new(c)) if n)
    return {"bytes": 2 * rows * (keys + new * c["n"]) + 2 * new * G * rows + keys // c["page"] * 4,
            "flops": 4 * H * G * D * (seen + new * c["n"])}


def _normal(shape, c, gen, std):
    return torch.empty(shape, dtype=_DTYPES[c["dtype"]], device="cuda").normal_(0.0, std, generator=gen)


def _pages(c, gen):
    """Page tensors, the table (pages in a shuffled order; -1: none) and the counts of tokens, as a server keeps them."""
    P, lens = c["page"], _lengths(c)
    need = [-(-l // P) for l in lens]
    total, width = sum(need) + 1, max(max(need), 1)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(gen.initial_seed() + 1)).int()
    table = torch.full((c["B"], width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (total, P, c["H"], c["D"])
    return {"cache_k": _normal(shape, c, gen, 0.5), "cache_v": _normal(shape, c, gen, 0.5), "table": table.cuda(),
            "past": torch.tensor(_past(c), dtype=torch.int32, device="cuda")}


def prepare(c, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    B, T, H, G, D = (c[x] for x in "BTHGD")
    s = {"case": c}
    if c["op"] == "rotary":
        s["q"], s["k"] = _normal((B, T * G, H, D), c, gen, 0.5), _normal((B, T, H, D), c, gen, 0.5)
        s["positions"] = torch.arange(c["lo"], c["lo"] + T, device="cuda")
        if c["grad"]:
            s["dq"], s["dk"] = _normal((B, T * G, H, D), c, gen, 1.0), _normal((B, T, H, D), c, gen, 1.0)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
    else:
        s.update(_pages(c, gen))
        new = _new(c)
    if c["op"] == "append":
        if c["ragged"]:
            b, t = 1, sum(new)
            s["cu"] = torch.tensor([0] + new).cumsum(0).int().cuda()
        else:
            b, t = B, T
        s["k"], s["v"] = _normal((b, t, H, D), c, gen, 0.5), _normal((b, t, H, D), c, gen, 0.5)
        s["q"] = _normal((b, t * G, H, D), c, gen, 0.5) if c["rot"] else None
        if c["L"]:
            s["depth_k"], s["depth_v"] = _normal((b, t * c["L"], H, D), c, gen, 0.5), _normal((b, t * c["L"], H, D), c, gen, 0.5)
    if c["op"] == "attend":
        s["q"] = _normal((B, T, H * G, D) if c["plain"] else (B, T * G, H, D), c, gen, 0.5)
        if c["ragged"]:
            s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        if c["L"]:
            s["depth_k"], s["depth_v"] = _normal((B, T * c["L"], H, D), c, gen, 0.5), _normal((B, T * c["L"], H, D), c, gen, 0.5)
    if c["rot"]:
        f, s["amplitude"] = _rates(c)
        s["rates"] = f.cuda()
        if own:
            import moda_amd

            scaling = None if c["scaling"] == "none" else c["scaling"]
            s["rotary"] = moda_amd.Rotary(c["rot"], base=_BASE, interleaved=c["pairs"] == "inter", scaling=scaling,
                                          factor=c["factor"], original_length=c["orig"] or None)
    return s


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import moda_amd

    c = s["case"]
    if c["op"] == "rotary":
        q, k = moda_amd.apply_rotary(s["q"], s["k"], s["rotary"], positions=s["positions"], moda_group_num=c["G"])
        if not c["grad"]:
            return [q, k]
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return [q.detach(), k.detach(), dq, dk]
    if c["op"] == "append":
        q = moda_amd.paged_append(s["k"], s["v"], s["cache_k"], s["cache_v"], s["table"], s["past"], cu_seqlens=s.get("cu"),
                                  q=s["q"], rotary=s.get("rotary"), moda_group_num=c["G"], cached_k=s.get("depth_k"),
                                  cached_v=s.get("depth_v"), depth_slot=c["n"])
        return [x for x in (s["cache_k"], s["cache_v"], q, s.get("depth_k"), s.get("depth_v")) if x is not None]
    if c["plain"]:
        return moda_amd.paged_attn(s["q"], s["cache_k"], s["cache_v"], s["table"], s["past"], new_lens=s.get("new"))
    return moda_amd.paged_moda(s["q"], s["cache_k"], s["cache_v"], s["table"], s["past"], new_lens=s.get("new"),
                               cached_k=s.get("depth_k"), cached_v=s.get("depth_v"), depth_valid=c["n"] or None,
                               moda_group_num=c["G"])


def _angles(s, positions):
    """cos, sin [..., pairs] of positions [...]: angles in 64 bits, whole turns taken off, the rest in 32."""
    turns = positions.double()[..., None] * s["rates"]
    a = ((turns - turns.round()) * (2 * math.pi)).float()
    return a.cos() * s["amplitude"], a.sin() * s["amplitude"]


def _rotated(c, x, cos, sin):
    """x [..., D] turned by the angles of its row, [..., pairs]."""
    R = c["rot"]
    head, rest = x[..., :R].float(), x[..., R:].float()
    if c["pairs"] == "half":
        a, b = head[..., :R // 2], head[..., R // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        y = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)
    return y.to(x.dtype)


def _run_plain(s):
    c = s["case"]
    with torch.no_grad():
        return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[c["op"]](s, c)


def _rows(cs, G):
    """Angles per token [..., T, pairs] -> per query row and head [..., T * G, 1, pairs]."""
    return [x.repeat_interleave(G, -2).unsqueeze(-2) for x in cs]


def _plain_rotary(s, c):
    cs = _angles(s, s["positions"])
    q, k = _rotated(c, s["q"], *_rows(cs, c["G"])), _rotated(c, s["k"], *_rows(cs, 1))
    if not c["grad"]:
        return [q, k]
    back = (cs[0], -cs[1])
    return [q, k, _rotated(c, s["dq"], *_rows(back, c["G"])), _rotated(c, s["dk"], *_rows(back, 1))]


def _plain_append(s, c):
    k, v, past = s["k"], s["v"], s["past"].long()
    if "cu" in s:
        cu = s["cu"].long()
        t = torch.arange(k.shape[1], device="cuda")
        b = torch.searchsorted(cu, t, right=True) - 1
        pos, b = (past[b] + t - cu[b])[None], b[None]
    else:
        pos = past[:, None] + torch.arange(k.shape[1], device="cuda")
        b = torch.arange(k.shape[0], device="cuda")[:, None].expand_as(pos)
    q = s["q"]
    if c["rot"]:
        cs = _angles(s, pos)
        k, q = _rotated(c, k, *_rows(cs, 1)), _rotated(c, q, *_rows(cs, c["G"]))
    page = s["table"].long()[b, pos // c["page"]]
    s["cache_k"][page, pos % c["page"]] = k
    s["cache_v"][page, pos % c["page"]] = v
    out = [s["cache_k"], s["cache_v"]] + ([q] if q is not None else [])
    if c["L"]:
        for name, x in (("depth_k", k), ("depth_v", v)):
            s[name].view(k.shape[0], k.shape[1], c["L"], c["H"], c["D"])[:, :, c["n"]] = x
            out.append(s[name])
    return out


def _plain_attend(s, c):
    B, T, H, G, D = (c[x] for x in "BTHGD")
    table, past = s["table"].long(), s["past"].long()
    S = table.shape[1] * c["page"]

    def heads(x):  # pages or depth slots [B, keys, H, D] -> [B, H, keys, D]
        return x.float().transpose(1, 2)

    k = heads(s["cache_k"][table.clamp(min=0)].reshape(B, S, H, D))
    if c["plain"]:
        q = s["q"].float().view(B, T, H, G, D).permute(0, 2, 1, 3, 4)
    else:
        q = s["q"].float().view(B, T, G, H, D).permute(0, 3, 1, 2, 4)
    q = q.reshape(B, H, T * G, D) * D ** -0.5
    logits = torch.matmul(q, k.transpose(-1, -2))
    del k
    token = torch.arange(T, device="cuda").repeat_interleave(G)
    seen = torch.arange(S, device="cuda") <= (past[:, None] + token)[..., None]
    if "new" in s:
        seen = seen & (token < s["new"][:, None])[..., None]
    logits = logits.masked_fill(~seen[:, None], -math.inf)
    n, L = c["n"], c["L"]
    if L:
        own_k, own_v = (heads(s[x].view(B, T, L, H, D)[:, :, :n].reshape(B, T * n, H, D)) for x in ("depth_k", "depth_v"))
        mine = token[:, None] == torch.arange(T, device="cuda").repeat_interleave(n)
        mine = mine.expand(B, -1, -1)
        if "new" in s:
            mine = mine & (token < s["new"][:, None])[..., None]
        logits = torch.cat([logits, torch.matmul(q, own_k.transpose(-1, -2)).masked_fill(~mine[:, None], -math.inf)], -1)
    top = logits.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (logits - top).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    v = heads(s["cache_v"][table.clamp(min=0)].reshape(B, S, H, D))
    o = torch.matmul(p[..., :S], v)
    if L:
        o = o + torch.matmul(p[..., S:], own_v)
    o = o.view(B, H, T, G, D)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, T, H * G, D) if c["plain"] else o.permute(0, 2, 3, 1, 4).reshape(B, T * G, H, D)
    return o.to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------------


def _turn(c, x, positions, back=False):
    """Rows x [..., H, D] at positions [...]: each pair as a complex number times amplitude * exp(i angle)."""
    f, amplitude = _rates(c)
    turns = torch.remainder(positions.double()[..., None] * f.to(positions.device), 1.0) * (2 * math.pi)
    w = torch.polar(torch.full_like(turns, amplitude), -turns if back else turns)[..., None, :]
    R, y = c["rot"], x.double().clone()
    first, second = (slice(0, R // 2), slice(R // 2, R)) if c["pairs"] == "half" else (slice(0, R, 2), slice(1, R, 2))
    z = torch.complex(y[..., first], y[..., second]) * w
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    c = case
    with torch.no_grad():
        s = prepare(c, seed)
        return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[c["op"]](s, c)


def _exact_rotary(s, c):
    per_row = s["positions"].repeat_interleave(c["G"])
    out = [_turn(c, s["q"], per_row), _turn(c, s["k"], s["positions"])]
    if c["grad"]:
        out += [_turn(c, s["dq"], per_row, back=True), _turn(c, s["dk"], s["positions"], back=True)]
    return out


def _exact_append(s, c):
    P, G, table = c["page"], c["G"], s["table"].tolist()
    ck, cv = s["cache_k"].double(), s["cache_v"].double()
    q = None if s["q"] is None else s["q"].double()
    depth = [s[x].double() for x in ("depth_k", "depth_v")] if c["L"] else []
    at = 0
    for b, (past, n) in enumerate(zip(_past(c), _new(c))):
        row, first = (0, at) if c["ragged"] else (b, 0)
        at += n
        if n == 0:
            continue
        pos = torch.arange(past, past + n, device="cuda")
        k, v = s["k"][row, first:first + n].double(), s["v"][row, first:first + n].double()
        if c["rot"]:
            k = _turn(c, k, pos)
            q[row, first * G:(first + n) * G] = _turn(c, q[row, first * G:(first + n) * G], pos.repeat_interleave(G))
        for page in range(past // P, (past + n - 1) // P + 1):
            i0, i1 = max(page * P, past), min((page + 1) * P, past + n)
            ck[table[b][page], i0 - page * P:i1 - page * P] = k[i0 - past:i1 - past]
            cv[table[b][page], i0 - page * P:i1 - page * P] = v[i0 - past:i1 - past]
        for x, y in zip(depth, (k, v)):
            x[row, c["n"]::c["L"]][:n] = y
    return [ck, cv] + ([q] if q is not None else []) + depth


def _exact_attend(s, c):
    T, H, G, D, P = c["T"], c["H"], c["G"], c["D"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    table = s["table"].tolist()
    for b, (past, n) in enumerate(zip(_past(c), _new(c))):
        if n == 0:
            continue
        pages = torch.tensor(table[b][:-(-(past + n) // P)], device="cuda")
        K, V = (s[x][pages].reshape(-1, H, D) for x in ("cache_k", "cache_v"))
        for t in range(n):
            for h in range(H):
                k, v = K[:past + t + 1, h].double(), V[:past + t + 1, h].double()
                if c["L"]:
                    k = torch.cat([k, s["depth_k"][b, t * c["L"]:t * c["L"] + c["n"], h].double()])
                    v = torch.cat([v, s["depth_v"][b, t * c["L"]:t * c["L"] + c["n"], h].double()])
                rows = (b, t, slice(h * G, (h + 1) * G)) if c["plain"] else (b, slice(t * G, (t + 1) * G), h)
                x = s["q"][rows].double() @ k.T / math.sqrt(D)
                out[rows] = torch.softmax(x, -1) @ v
    return out
