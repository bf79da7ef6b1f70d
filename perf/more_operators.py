"""The operators of a language model's training step around the recurrence, as measurable cases: the
embedding of tokens with its gradient, the log probabilities of given tokens with entropy, the top
alternatives and the gradient, the choice of units with its balance loss and gradient, and the
gradients' global norm with clipping. Each case is a dict of sizes and options; :func:`prepare`
makes what a program holds before the call, :func:`run` is one pass, :func:`exact` the same values in
64 bits.

``own`` chooses what :func:`run` calls: the operators written out in elementary torch operations,
or the package's own.
"""

from __future__ import annotations

import math

import torch

own = False

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
F64 = torch.float64

#: the tensor sizes of the lists whose gradients are clipped, besides "ragged"
LISTS = {
    # a recurrent model's 198 weights, 1.97 M elements
    "model": [64 * 64] * 48 + [256 * 64] * 96 + [64] * 48 + [256 * 128] * 6,
    # 64 weights of 4 M elements
    "large": [1 << 22] * 64,
}


def listed():
    return [
        # one decoded token of every sequence of a small batch, some of them padding
        dict(name="embed_step", kind="embed", B=32, T=1, V=32000, D=2048, table="bf16", out="bf16",
             scale=1.0, padded=True),
        # odd sizes in half precision, the cotangent a slice of a wider product's
        dict(name="embed_odd", kind="embed_train", B=3, T=1021, V=5003, D=100, table="f16",
             out="f16", scale=10.0, padded=True),
        # a training window of the reference shape's rows and positions: fp32 weights, bf16 activations
        dict(name="embed_window", kind="embed_train", B=32, T=256, V=32000, D=512, table="f32",
             out="bf16", scale=1.0, padded=False),
        # a long training window over a large vocabulary
        dict(name="embed_long", kind="embed_train", B=8, T=4096, V=131072, D=2048, table="bf16",
             out="bf16", scale=45.25, padded=False),
        # one answered token with its most probable alternatives
        dict(name="score_one", kind="score", n=1, V=32000, io="bf16", top=20, skipped=False),
        # a prompt's tokens scored over a large odd vocabulary
        dict(name="score_prompt", kind="score", n=1000, V=131071, io="bf16", top=5, skipped=False),
        # a training window's loss with an entropy bonus, fp32 logits, an odd vocabulary, padded rows
        dict(name="score_odd", kind="score_train", n=301, V=50021, io="f32", entropy=True,
             skipped=True),
        # a training window's loss, the reference shape's rows and positions
        dict(name="score_window", kind="score_train", n=8192, V=32000, io="bf16", entropy=False,
             skipped=True),
        # a training window through the model's own unit bank
        dict(name="route_model", kind="route", n=8192, M=8, k=2, io="f32", padded=False),
        # a long training window through a layer of many units, padded rows
        dict(name="route_long", kind="route", n=65536, M=64, k=8, io="bf16", padded=True),
        # the clip of a small model's 198 gradients
        dict(name="clip_model", kind="clip", sizes="model", io="f32", count=198),
        # the clip of large gradients
        dict(name="clip_large", kind="clip", sizes="large", io="f32", count=64),
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng, lo, hi):
    """A width: often a common one, else any, half of these even to eight elements."""
    if rng.random() < 0.5:
        return rng.choice([w for w in (64, 96, 128, 192, 256, 384, 512, 640, 768, 1024, 1280, 2048,
                                       2560, 4096) if lo <= w <= hi])
    return max(lo, _log(rng, lo, hi) // (step := rng.choice([8, 1])) * step)


def draw(rng):
    kind = rng.choice(["embed", "embed_train", "embed_train", "score", "score_train", "score_train",
                       "route", "route", "clip", "clip"])
    io = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind in ("embed", "embed_train"):
        while True:
            case = dict(kind=kind, B=_log(rng, 1, 64), T=_log(rng, 1, 8192), V=_log(rng, 100, 262144),
                        D=_width(rng, 32, 4096), table=io, out=rng.choice([io, io, "bf16"]),
                        scale=rng.choice([1.0, 0.5, 22.625]), padded=rng.random() < 0.5)
            if case["B"] * case["T"] <= 65536 and work(case)["bytes"] <= 9e8:
                return case
    if kind in ("score", "score_train"):
        while True:
            n, V = _log(rng, 1, 16384), _log(rng, 500, 262144)
            if n * V * SIZE[io] <= 8192 * 32000 * 2:
                break
        if kind == "score":
            return dict(kind=kind, n=n, V=V, io=io, top=rng.choice([0, 1, 5, 20]),
                        skipped=rng.random() < 0.25)
        return dict(kind=kind, n=n, V=V, io=io, entropy=rng.random() < 0.5,
                    skipped=rng.random() < 0.5)
    if kind == "route":
        while True:
            n, M = _log(rng, 1, 131072), _log(rng, 4, 256)
            if n * M <= 2 ** 24:
                return dict(kind=kind, n=n, M=M, k=rng.randint(1, min(8, M)), io=io,
                            padded=rng.random() < 0.5)
    count = _log(rng, 1, 600)
    return dict(kind=kind, sizes="ragged", io=rng.choice([io, "mixed"]) if count > 2 else io,
                count=count)


# ------------------------------------------------------------------------------------------
# Inputs.
# ------------------------------------------------------------------------------------------

def _ragged(count, seed):
    """Sizes from one element to a million, the small ones many."""
    g = torch.Generator().manual_seed(seed)
    return [int(v) for v in (2.0 ** (20 * torch.rand(count, generator=g) ** 1.5)).tolist()]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def rnd(*shape, scale=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    kind = case["kind"]
    if kind in ("embed", "embed_train"):
        B, T, V, D = (case[k] for k in ("B", "T", "V", "D"))
        # the r-th most frequent token has a share of about 1 / r
        rank = (torch.exp(uniform(B, T).double() * math.log(V + 1.0)).long() - 1).clamp_(0, V - 1)
        tokens = torch.randperm(V, generator=g, device="cuda")[rank]
        if case["padded"]:  # rows end at places of their own, then there is padding
            end = (uniform(B, 1) * 1.25 * T).ceil()
            tokens = torch.where(torch.arange(T, device="cuda") < end, tokens, -1)
        s.update(tokens=tokens, weight=rnd(V, D, scale=D ** -0.5, dtype=IO[case["table"]]))
        if kind == "embed_train":
            wide = rnd(B, T, 2 * D if case["padded"] else D, dtype=IO[case["out"]])
            s["d_out"] = wide[..., :D]
    elif kind in ("score", "score_train"):
        n, V = case["n"], case["V"]
        # a peaked distribution over a common background, the vocabulary's last entries masked
        logits = rnd(V, scale=1.5) + rnd(n, V, scale=2.0)
        logits[:, V - V // 100:] = float("-inf")
        logits = logits.to(IO[case["io"]])
        live = V - V // 100
        tokens = torch.where(uniform(n) < 0.5, logits.argmax(dim=1), (uniform(n) * live).long())
        if case["skipped"]:
            tokens = torch.where(uniform(n) < 1 / 8, -1, tokens)
        s.update(logits=logits, tokens=tokens)
        if kind == "score_train":
            s["d_logprob"] = -uniform(n) / n
            s["d_entropy"] = rnd(n, scale=0.01 / n) if case["entropy"] else None
    elif kind == "route":
        n, M, k = case["n"], case["M"], case["k"]
        logits = rnd(M, scale=0.5) + rnd(n, M)
        s.update(logits=logits.to(IO[case["io"]]), valid=None, d_shares=rnd(n, k, scale=0.1),
                 d_balance=torch.full((), 0.01, device="cuda") * (1.0 + uniform(1)[0]))
        if case["padded"]:
            s["valid"] = uniform(n) < 7 / 8
    else:
        sizes = LISTS.get(case["sizes"]) or _ragged(case["count"], case["count"])
        types = [IO[case["io"]]] if case["io"] != "mixed" else list(IO.values())
        grads, out, flat = [], [], []
        for i, t in enumerate(types):
            mine = sizes[i::len(types)]
            # what is clipped goes to one buffer a type, tensor after tensor
            flat.append(torch.zeros(sum(mine), dtype=t, device="cuda"))
            grads += [rnd(m, scale=0.01, dtype=t) for m in mine]
            out += list(flat[-1].split(mine))
        # the norm is about 0.01 sqrt(elements): a third of it is left
        s.update(grads=grads, out=out, flat=flat, max_norm=0.01 * math.sqrt(sum(sizes)) / 3)
    return s


# ------------------------------------------------------------------------------------------
# One pass.
# ------------------------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)[s["kind"]](s)


def _plain_rows(s):
    """The tokens with padding as row ``V``."""
    return torch.where((s["tokens"] >= 0) & (s["tokens"] < s["V"]), s["tokens"], s["V"])


def _plain_embed(s):
    rows = _plain_rows(s)
    taken = s["weight"][rows.clamp(max=s["V"] - 1)].float() * s["scale"]
    return {"out": torch.where((rows < s["V"])[..., None], taken, 0.0).to(IO[s["out"]])}


def _plain_embed_train(s):
    d = s["d_out"].float().reshape(-1, s["D"]) * s["scale"]
    sums = torch.zeros(s["V"] + 1, s["D"], device=d.device)
    sums.index_add_(0, _plain_rows(s).reshape(-1), d)
    return {**_plain_embed(s), "d_table": sums[:-1].to(s["weight"].dtype)}


def _plain_logprobs(s):
    """The rows' log probabilities, probabilities, and entropy."""
    x = s["logits"].float()
    x = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(dim=1, keepdim=True)
    rest = torch.log(total)
    entropy = rest - torch.where(e > 0, e * x, 0.0).sum(dim=1, keepdim=True) / total
    return x - rest, e / total, entropy[:, 0]


def _plain_given(s, logp):
    given = (s["tokens"] >= 0) & (s["tokens"] < s["V"])
    at = torch.where(given, s["tokens"], 0)[:, None]
    return given, at, torch.where(given, logp.gather(1, at)[:, 0], 0.0)


def _plain_score(s):
    logp, _, entropy = _plain_logprobs(s)
    out = {"logprob": _plain_given(s, logp)[2], "entropy": entropy}
    if s["top"]:
        order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True).indices
        best = order[:, :s["top"]]
        out.update(top_tokens=best, top_logprobs=logp.gather(1, best))
    return out


def _plain_score_train(s):
    logp, p, entropy = _plain_logprobs(s)
    given, at, logprob = _plain_given(s, logp)
    g = torch.where(given, s["d_logprob"], 0.0)[:, None]
    d = -g * p
    if s["d_entropy"] is not None:
        d = d - torch.where(p > 0, s["d_entropy"][:, None] * p * (logp + entropy[:, None]), 0.0)
    d.scatter_add_(1, at, g)
    return {"logprob": logprob, "entropy": entropy, "d_logits": d.to(s["logits"].dtype)}


def _plain_route(s):
    x = s["logits"].float()
    n, M = x.shape
    live = torch.ones(n, 1, device=x.device) if s["valid"] is None else s["valid"][:, None].float()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    units = torch.where(live > 0, order.indices[:, :s["k"]], -1)
    e = torch.exp(order.values[:, :s["k"]] - order.values[:, :1])
    shares = live * e / e.sum(dim=1, keepdim=True)
    p = torch.exp(x - order.values[:, :1])
    p = live * p / p.sum(dim=1, keepdim=True)
    at = torch.arange(M, device=x.device)
    chosen = (units[..., None] == at).any(dim=1)
    counts = chosen.sum(dim=0)
    load = counts.double() / counts.sum().clamp(min=1)
    rows = live.double().sum().clamp(min=1)
    probs = p.sum(dim=0, dtype=F64) / rows
    balance = M * (load * probs).sum()
    # the shares' gradient at the chosen units, and the balance's through the probabilities
    d_s = shares * (s["d_shares"] - (shares * s["d_shares"]).sum(dim=1, keepdim=True))
    d = torch.zeros_like(x).scatter_add_(1, units.clamp(min=0), d_s)
    load = load.float()
    d = d + s["d_balance"] * (M / rows.float()) * p * (load - (p * load).sum(dim=1, keepdim=True))
    return {"units": units, "shares": shares, "counts": counts, "probs": probs.float(),
            "balance": balance.float(), "d_logits": d.to(s["logits"].dtype)}


def _plain_clip(s):
    grads = torch.cat([g.double() for g in s["grads"]])
    norm = torch.sqrt((grads * grads).sum()).reshape(1)
    coefficient = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    scaled = (grads * coefficient).split([f.numel() for f in s["flat"]])
    return {"norm": norm, "coefficient": coefficient,
            "grads": [f.copy_(t.float()) for f, t in zip(s["flat"], scaled)]}


_plain = {"embed": _plain_embed, "embed_train": _plain_embed_train, "score": _plain_score,
          "score_train": _plain_score_train, "route": _plain_route, "clip": _plain_clip}


def _own_embed(s):
    from hsn_amd import embedding

    return {"out": embedding.forward(s["tokens"], s["weight"], scale=s["scale"], dtype=IO[s["out"]])}


def _own_embed_train(s):
    from hsn_amd import embedding

    return {**_own_embed(s),
            "d_table": embedding.backward(s["tokens"], s["d_out"], s["V"], scale=s["scale"],
                                          dtype=s["weight"].dtype)}


def _own_score(s):
    from hsn_amd import scoring

    out = scoring.forward(s["logits"], s["tokens"], top=s["top"], save=False)
    names = ("logprob", "entropy", "top_tokens", "top_logprobs")
    return {name: out[name] for name in names[:4 if s["top"] else 2]}


def _own_score_train(s):
    from hsn_amd import scoring

    out = scoring.forward(s["logits"], s["tokens"])
    d_logits = scoring.backward(s["logits"], s["tokens"], out["stats"], s["d_logprob"],
                                s["d_entropy"])
    return {"logprob": out["logprob"], "entropy": out["entropy"], "d_logits": d_logits}


def _own_route(s):
    from hsn_amd import unit_router

    out = unit_router.forward(s["logits"], s["k"], valid=s["valid"])
    d_logits = unit_router.backward(s["logits"], out["units"], out["tally"], s["d_shares"],
                                    s["d_balance"], valid=s["valid"])
    return {"units": out["units"], "shares": out["shares"], "counts": out["counts"],
            "probs": out["probs"], "balance": out["balance"], "d_logits": d_logits}


def _own_clip(s):
    from hsn_amd import grad_clip

    norm, coefficient = grad_clip.clip(s["grads"], s["max_norm"], out=s["out"])
    return {"norm": norm, "coefficient": coefficient, "grads": s["flat"]}


_own = {"embed": _own_embed, "embed_train": _own_embed_train, "score": _own_score,
        "score_train": _own_score_train, "route": _own_route, "clip": _own_clip}


# ------------------------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits.
# ------------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("embed", "embed_train"):
        n, V, D = case["B"] * case["T"], case["V"], case["D"]
        if case["padded"]:
            n = int(0.6 * n) + 1  # the mean share of live positions
        share = torch.arange(1, V + 1, dtype=F64)
        share = torch.log1p(1.0 / share) / math.log(V + 1.0)
        rows = float(-torch.expm1(n * torch.log1p(-share)).sum())  # different tokens, on average
        st, so = SIZE[case["table"]], SIZE[case["out"]]
        tokens = 8 * case["B"] * case["T"]
        work = {"bytes": tokens + rows * D * st + case["B"] * case["T"] * D * so, "flops": n * D}
        if kind == "embed_train":
            work = {"bytes": work["bytes"] + n * D * so + V * D * st, "flops": 3 * n * D}
        return work
    if kind in ("score", "score_train"):
        n, V, size = case["n"], case["V"], SIZE[case["io"]]
        if kind == "score":
            return {"bytes": n * (V * size + 16 + 12 * case["top"]), "flops": 6 * n * V}
        return {"bytes": n * (2 * V * size + 24), "flops": 12 * n * V}
    if kind == "route":
        n, M, k = case["n"], case["M"], case["k"]
        return {"bytes": n * (2 * M * SIZE[case["io"]] + 16 * k) + 12 * M,
                "flops": n * (10 * M + k * M)}
    sizes = LISTS.get(case["sizes"]) or _ragged(case["count"], case["count"])
    types = [case["io"]] if case["io"] != "mixed" else list(IO)
    return {"bytes": sum(2 * SIZE[t] * sum(sizes[i::len(types)]) for i, t in enumerate(types)),
            "flops": 3 * sum(sizes)}


def exact(case, seed):
    """The operators' definitions in 64 bits, rows at a time where they are long; whole numbers have
    no such value."""
    kind = case["kind"]
    s = prepare(case, seed)
    if kind in ("embed", "embed_train"):
        V, D = case["V"], case["D"]
        flat = s["tokens"].reshape(-1)
        at = torch.nonzero(flat >= 0)[:, 0]
        out = torch.zeros(flat.numel(), D, dtype=F64, device=flat.device)
        out[at] = s["weight"].index_select(0, flat[at]).to(F64) * case["scale"]
        values = {"out": out.view(*s["tokens"].shape, D)}
        if kind == "embed_train":
            d = s["d_out"].reshape(-1, D)[at].to(F64)
            sums = torch.zeros(V, D, dtype=F64, device=d.device)
            sums.index_put_((flat[at],), d, accumulate=True)
            values["d_table"] = sums * case["scale"]
        return values
    if kind in ("score", "score_train"):
        n, V = case["n"], case["V"]
        logprob = torch.zeros(n, dtype=F64, device="cuda")
        entropy = torch.zeros(n, dtype=F64, device="cuda")
        top = torch.zeros(n, case.get("top", 0), dtype=F64, device="cuda")
        grad = torch.zeros(n, V, dtype=F64, device="cuda") if kind == "score_train" else None
        for i in range(0, n, 512):
            rows = slice(i, min(n, i + 512))
            l = s["logits"][rows].to(F64)
            l = l - torch.logsumexp(l, dim=1, keepdim=True)
            p = torch.exp(l)
            entropy[rows] = -torch.special.xlogy(p, p).sum(dim=1)
            token = s["tokens"][rows]
            have = torch.nonzero(token >= 0)[:, 0]
            logprob[rows.start + have] = l[have, token[have]]
            if kind == "score":
                top[rows] = torch.topk(l, case["top"], dim=1).values
                continue
            d = torch.zeros_like(l)
            if s["d_entropy"] is not None:
                d = -s["d_entropy"][rows].to(F64)[:, None] * (
                    torch.special.xlogy(p, p) + p * entropy[rows][:, None])
            g = s["d_logprob"][rows].to(F64)[have]
            d[have] -= g[:, None] * p[have]
            d[have, token[have]] += g
            grad[rows] = d
        values = {"logprob": logprob, "entropy": entropy}
        if kind == "score_train":
            values["d_logits"] = grad
        elif case["top"]:
            values.update(top_tokens=None, top_logprobs=top)
        return values
    if kind == "route":
        l = s["logits"].to(F64).requires_grad_()
        n, M = l.shape
        rows = torch.arange(n, device=l.device) if s["valid"] is None else torch.nonzero(s["valid"])[:, 0]
        # the chosen units: those with fewer than k units before them
        x = l.detach()
        before = torch.zeros(n, M, dtype=torch.int64, device=l.device)
        at = torch.arange(M, device=l.device)
        for j in range(M):
            before += (x[:, j:j + 1] > x) | ((x[:, j:j + 1] == x) & (j < at))
        units = torch.zeros(n, case["k"], dtype=torch.int64, device=l.device)
        for j in range(case["k"]):
            units[:, j] = torch.nonzero(before == j)[:, 1]
        shares = torch.zeros(n, case["k"], dtype=F64, device=l.device)
        shares = shares.index_put((rows,), torch.softmax(l.gather(1, units)[rows], dim=1))
        load = torch.bincount(units[rows].reshape(-1), minlength=M).to(F64)
        load = load / max(1.0, float(load.sum()))
        probs = torch.softmax(l[rows], dim=1).sum(dim=0) / max(1, rows.numel())
        balance = M * (load * probs).sum()
        loss = (shares * s["d_shares"].to(F64)).sum() + s["d_balance"].to(F64) * balance
        d, = torch.autograd.grad(loss, l)
        return {"units": None, "shares": shares.detach(), "counts": None, "probs": probs.detach(),
                "balance": balance.detach(), "d_logits": d}
    squares = sum(float(torch.dot(g.to(F64), g.to(F64))) for g in s["grads"])
    norm = math.sqrt(squares)
    coefficient = min(1.0, s["max_norm"] / (norm + 1e-6))
    flat, i = [], 0
    for f in s["flat"]:
        parts, have = [], 0
        while have < f.numel():
            parts.append(s["grads"][i].to(F64) * coefficient)
            have, i = have + parts[-1].numel(), i + 1
        flat.append(torch.cat(parts) if parts else f.to(F64))
    one = torch.ones(1, dtype=F64)
    return {"norm": norm * one, "coefficient": coefficient * one, "grads": flat}
