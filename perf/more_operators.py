"""The two ends of a language model, tokens to rows and rows to a loss over the vocabulary: what is measured, as plain torch
operations (``own = False``) and as calls of this package's kernels (``own = True``).

  op      embed  ``embed_tokens`` (``grad``: with the gradient of the weight)
          loss   ``linear_cross_entropy`` (``grad``: with the gradients of the rows and the weight)
  dtype   bf16 | fp16 | fp32
  B, T    sequences, tokens of each;  V: words of the vocabulary;  C: width of a row
  scale   on the rows (``embed``) or on the logits (``loss``)
  none    per cent of the tokens that are no word (``embed``: padding) or have no target (``loss``)
  reduce  mean | sum | none (``none`` with ``grad``: every row's loss has an upstream gradient of its own)

Words are drawn with a probability of about one over their rank, as in text.  Rows are N(0, 1), as behind a norm, plus a share of
their target's own weight, so that some targets are likely and others are not; weights are N(0, 1/C).
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_IGNORED = -100


def _case(op, B, T, V, C, dtype="bf16", grad=False, scale=1.0, none=0, reduce="none"):
    return {"op": op, "B": B, "T": T, "V": V, "C": C, "dtype": dtype, "grad": grad, "scale": scale, "none": none, "reduce": reduce}


def listed():
    cases = {
        # the row of one generated token: a launch and the host time of the call are all of it
        "embed-token": _case("embed", 1, 1, 32000, 2048),
        # the long-context training step, forward and backward, a large vocabulary
        "embed-64k-train": _case("embed", 1, 65536, 131072, 2048, grad=True),
        # fp32 fine-tuning of a small model on padded sequences, odd sizes, rows scaled by the root of the width
        "embed-padded-train": _case("embed", 3, 1021, 50257, 384, "fp32", grad=True, scale=math.sqrt(384), none=30),
        # the log-likelihood of one token
        "loss-token": _case("loss", 1, 1, 32000, 2048),
        # five drafted tokens of sixteen sequences to be scored
        "loss-drafts": _case("loss", 16, 5, 50257, 512, "fp16"),
        # a document is scored
        "loss-score": _case("loss", 1, 4096, 65536, 1024),
        # language-model training step at an ordinary context length
        "loss-4k-train": _case("loss", 2, 4096, 32000, 2048, grad=True, reduce="mean"),
        # the largest: long sequences on a large vocabulary
        "loss-16k-train": _case("loss", 1, 16384, 131072, 2048, grad=True, reduce="mean"),
        # training on answers alone: three of five rows are prompts and have no target
        "loss-answers-train": _case("loss", 5, 819, 50257, 768, "fp16", grad=True, none=60, reduce="mean"),
        # every row's loss weighted by the caller, a small vocabulary, sizes off the tiles, logits scaled
        "loss-weighted-train": _case("loss", 1, 509, 4099, 1000, grad=True, scale=0.5),
        # fp32: gradient checks and small models
        "loss-fp32-train": _case("loss", 1, 1021, 10007, 256, "fp32", grad=True, none=5, reduce="sum"),
    }
    return [dict(c, name=k) for k, c in cases.items()]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm, odd as often as even."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    top = work(next(c for c in listed() if c["name"] == "loss-16k-train"))
    while True:
        op = rng.choice(["embed", "loss", "loss"])
        T, V = _between(rng, 1, 32768), _between(rng, 300, 131072)
        C = rng.choice([64, 128, 256, 384, 512, 768, 1024, 2048, 4096, 8 * _between(rng, 8, 512), _between(rng, 64, 4096)])
        c = _case(op, rng.choice([1, 1, 2, 3, 8]), T, V, C, rng.choice(["bf16", "bf16", "fp16", "fp32"]), grad=rng.random() < 0.6,
                  scale=rng.choice([1.0, 1.0, 0.5, round(C ** 0.5, 3) if op == "embed" else 1.5]),
                  none=rng.choice([0, 0, rng.randint(1, 90)]), reduce=rng.choice(["mean", "mean", "sum", "none"]) if op == "loss" else "none")
        w = work(c)
        # in 32 bits the matrix instruction is slower: leave room for that
        if w["flops"] * (8 if c["dtype"] == "fp32" else 1) <= top["flops"] and w["bytes"] <= 2 * top["bytes"]:
            return c


def work(c):
    es, N, V, C = _SIZES[c["dtype"]], c["B"] * c["T"], c["V"], c["C"]
    live = _live(c)
    if c["op"] == "embed":
        back = live * C * es + V * C * es + 8 * N if c["grad"] else 0
        return {"bytes": (live + N) * C * es + 8 * N + back, "flops": 2 * live * C * (2 if c["grad"] else 1)}
    back = live * C * es + N * C * es + 2 * V * C * es if c["grad"] else 0
    return {"bytes": live * C * es + V * C * es + 12 * N + back, "flops": 2 * live * V * C * (3 if c["grad"] else 1)}


def _live(c):
    """Tokens that are words, or have a target: those whose place in a fixed order is not among the ``none`` per cent."""
    N = c["B"] * c["T"]
    return N - N * c["none"] // 100


def _words(c, gen):
    """Tokens [B, T]: word k with a probability of about 1 / (k + 1), a random choice of places without one."""
    N, V = c["B"] * c["T"], c["V"]
    u = torch.rand(N, generator=gen, device="cuda", dtype=torch.float64)
    t = ((V + 1.0) ** u).floor().long().clamp(1, V) - 1
    place = torch.rand(N, generator=gen, device="cuda").argsort()
    t[place[_live(c):]] = _IGNORED if c["op"] == "loss" else -1
    return t.view(c["B"], c["T"])


def prepare(c, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt, B, T, V, C = _DTYPES[c["dtype"]], c["B"], c["T"], c["V"], c["C"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(0.0, std, generator=gen)

    s = {"case": c, "tokens": _words(c, gen), "weight": normal(V, C, std=C ** -0.5)}
    if c["op"] == "embed":
        if c["grad"]:
            s["dy"] = normal(B, T, C)
    else:
        # the target's logit is raised by 0 .. 12
        raised = 12 * torch.rand(B, T, 1, generator=gen, device="cuda") / c["scale"]
        x = s["weight"][s["tokens"].clamp(min=0)].float() * raised
        s["x"] = x.normal_(0.0, 1.0, generator=gen).add_(s["weight"][s["tokens"].clamp(min=0)].float() * raised).to(dt)
        if c["grad"]:
            s["x"].requires_grad_()
            s["upstream"] = torch.rand((B, T) if c["reduce"] == "none" else (), generator=gen, device="cuda") + 0.5
    if c["grad"]:
        s["weight"].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import moda_amd

    c = s["case"]
    if c["op"] == "embed":
        y = moda_amd.embed_tokens(s["tokens"], s["weight"], scale=c["scale"])
        return [y.detach(), *torch.autograd.grad(y, s["weight"], s["dy"])] if c["grad"] else [y]
    loss = moda_amd.linear_cross_entropy(s["x"], s["weight"], s["tokens"], scale=c["scale"], ignore_index=_IGNORED,
                                         reduction=c["reduce"])
    return [loss.detach(), *torch.autograd.grad(loss, (s["x"], s["weight"]), s["upstream"])] if c["grad"] else [loss]


def _run_plain(s):
    c = s["case"]
    with torch.no_grad():
        return (_plain_embed if c["op"] == "embed" else _plain_loss)(s, c)


def _plain_embed(s, c):
    t, w = s["tokens"], s["weight"]
    word = ((t >= 0) & (t < c["V"]))[..., None]
    y = (w[t.clamp(0, c["V"] - 1)].float() * c["scale"]).masked_fill(~word, 0).to(w.dtype)
    if not c["grad"]:
        return [y]
    dy = (s["dy"].float() * c["scale"]).masked_fill(~word, 0)
    dw = torch.zeros(c["V"], c["C"], device="cuda").index_add_(0, t.clamp(0, c["V"] - 1).flatten(), dy.flatten(0, 1))
    return [y, dw.to(w.dtype)]


def _plain_loss(s, c):
    t = s["tokens"].flatten()
    live = ((t != _IGNORED) & (t >= 0) & (t < c["V"])).nonzero().flatten()
    x, w, t = s["x"].flatten(0, 1)[live].float(), s["weight"].float(), t[live]
    z = torch.matmul(x, w.T) * c["scale"]
    top = z.amax(-1, keepdim=True)
    lse = top + (z - top).exp().sum(-1, keepdim=True).log()
    rows = torch.zeros(c["B"] * c["T"], device="cuda")
    at = torch.arange(live.numel(), device="cuda")
    rows[live] = lse.flatten() - z[at, t]
    share = 1.0 / max(1, live.numel()) if c["reduce"] == "mean" else 1.0
    loss = rows.view(c["B"], c["T"]) if c["reduce"] == "none" else rows.sum() * share
    if not c["grad"]:
        return [loss]
    g = (s["upstream"].flatten()[live, None] if c["reduce"] == "none" else s["upstream"] * share) * c["scale"]
    dz = z.sub_(lse).exp_().mul_(g)
    dz[at, t] -= g.expand(live.numel(), 1).flatten()
    dx = torch.zeros(rows.numel(), c["C"], device="cuda")
    dx[live] = torch.matmul(dz, w)
    return [loss, dx.view(s["x"].shape).to(s["x"].dtype), torch.matmul(dz.T, x).to(s["weight"].dtype)]


# ------------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return (_exact_embed if case["op"] == "embed" else _exact_loss)(case, prepare(case, seed))


def _exact_embed(c, s):
    t = s["tokens"].flatten()
    y = torch.zeros(t.numel(), c["C"], dtype=torch.float64, device="cuda")
    words = (t >= 0).nonzero().flatten()
    y[words] = s["weight"][t[words]].double() * c["scale"]
    out = [y.view(c["B"], c["T"], c["C"])]
    if c["grad"]:
        # rows in the order of their words: the sum of a word's rows is the difference of two running sums
        word, order = t[words].sort(stable=True)
        dw = torch.zeros(c["V"], c["C"], dtype=torch.float64, device="cuda")
        seen, count = word.unique_consecutive(return_counts=True)
        last = count.cumsum(0)
        for c0 in range(0, c["C"], 256):
            total = s["dy"].flatten(0, 1)[words[order], c0:c0 + 256].double().cumsum(0)
            total = torch.cat([torch.zeros_like(total[:1]), total])
            dw[seen, c0:c0 + 256] = (total[last] - total[last - count]) * c["scale"]
        out.append(dw)
    return out


def _exact_loss(c, s):
    N, V, C, t = c["B"] * c["T"], c["V"], c["C"], s["tokens"].flatten()
    x, w = s["x"].detach().reshape(N, C), s["weight"].detach().double()
    live = (t >= 0).nonzero().flatten()
    rows = torch.zeros(N, dtype=torch.float64, device="cuda")
    dx = torch.zeros(N, C, dtype=torch.float64, device="cuda")
    dw = torch.zeros(V, C, dtype=torch.float64, device="cuda")
    share = 1.0 / max(1, live.numel()) if c["reduce"] == "mean" else 1.0
    step = max(1, 1 << 27 >> V.bit_length())
    for i in range(0, live.numel(), step):
        r = live[i:i + step]
        xr = x[r].double()
        log_p = torch.log_softmax(c["scale"] * (xr @ w.T), -1)
        rows[r] = -log_p.gather(1, t[r, None])[:, 0]
        if c["grad"]:
            g = s["upstream"].double().flatten()[r] if c["reduce"] == "none" else (s["upstream"].double() * share).expand(len(r))
            dz = (log_p.exp() - torch.nn.functional.one_hot(t[r], V)) * (g * c["scale"])[:, None]
            dx[r] = dz @ w
            dw += dz.T @ xr
    loss = rows.view(c["B"], c["T"]) if c["reduce"] == "none" else rows.sum() * share
    return [loss, dx.view(c["B"], c["T"], C), dw] if c["grad"] else [loss]
