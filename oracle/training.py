"""The training step's operators in float64 on the CPU, element by element: the embedding of tokens,
the log probabilities of given tokens, the choice of units with its balance, and the gradients' global
norm. Test infrastructure only."""

from __future__ import annotations

import math

import torch

F64 = torch.float64


def embed(tokens, table, scale=1.0):
    """``[..., D]``: the tokens' rows times ``scale``; a token outside the table gives zeros."""
    out = torch.zeros(tokens.numel(), table.shape[1], dtype=F64)
    for i, t in enumerate(tokens.reshape(-1).tolist()):
        if 0 <= t < table.shape[0]:
            out[i] = table[t].to(F64) * scale
    return out.reshape(*tokens.shape, table.shape[1])


def embed_backward(tokens, d_out, V, scale=1.0):
    """``[V, D]``: the sums of the tokens' cotangents times ``scale``, and the sums of their sizes."""
    D = d_out.shape[-1]
    d_table, size = torch.zeros(V, D, dtype=F64), torch.zeros(V, D, dtype=F64)
    for t, d in zip(tokens.reshape(-1).tolist(), d_out.reshape(-1, D).to(F64)):
        if 0 <= t < V:
            d_table[t] += d * scale
            size[t] += d.abs() * abs(scale)
    return d_table, size


def score(logits, tokens, top=0):
    """``(logprob [n], entropy [n], top tokens [n, top], their log probabilities)``."""
    n, V = logits.shape
    logprob, entropy = torch.zeros(n, dtype=F64), torch.zeros(n, dtype=F64)
    best = torch.full((n, top), -1, dtype=torch.int64)
    best_logprob = torch.full((n, top), -math.inf, dtype=F64)
    for i in range(n):
        row = logits[i].to(F64)
        t = int(tokens[i])
        given = 0 <= t < V
        if bool(row.isnan().any()) or bool((row == math.inf).any()):
            entropy[i] = math.nan
            logprob[i] = math.nan if given else 0.0
        elif bool((row == -math.inf).all()):
            logprob[i] = -math.inf if given else 0.0
        else:
            x = row - row.max()
            rest = torch.log(torch.exp(x).sum())
            logp = x - rest
            p = torch.exp(logp)
            entropy[i] = -torch.where(p > 0, p * logp, 0.0).sum()
            logprob[i] = logp[t] if given else 0.0
        fine = torch.nonzero(row > -math.inf)[:, 0]  # (not NaN either)
        order = fine[torch.sort(-row[fine], stable=True).indices][:top].tolist()
        for r, j in enumerate(order):
            best[i, r] = j
            best_logprob[i, r] = math.nan if math.isnan(float(entropy[i])) else logp[j]
    return logprob, entropy, best, best_logprob


def score_backward(logits, tokens, d_logprob, d_entropy=None):
    """``d_logits [n, V]`` by the formulas."""
    n, V = logits.shape
    _, entropy, _, _ = score(logits, tokens)
    d = torch.zeros(n, V, dtype=F64)
    for i in range(n):
        row = logits[i].to(F64)
        if bool((row == -math.inf).all()):
            continue
        if math.isnan(float(entropy[i])):
            d[i] = math.nan
            continue
        logp = torch.log_softmax(row, dim=0)
        p = torch.exp(logp)
        t = int(tokens[i])
        if 0 <= t < V and d_logprob is not None:
            d[i] -= p * float(d_logprob[i])
            d[i, t] += float(d_logprob[i])
        if d_entropy is not None:
            d[i] -= torch.where(p > 0, p * (logp + entropy[i]), 0.0) * float(d_entropy[i])
    return d


def choose_units(logits, k, valid=None):
    """``(units [n, k], shares [n, k], balance, counts [M], probs [M], rows)``."""
    n, M = logits.shape
    units, shares = torch.full((n, k), -1, dtype=torch.int64), torch.zeros(n, k, dtype=F64)
    counts, probs, rows = torch.zeros(M, dtype=torch.int64), torch.zeros(M, dtype=F64), 0
    for i in range(n):
        row = logits[i].to(F64)
        values = [math.inf if math.isnan(v) else v for v in row.tolist()]
        order = sorted((j for j in range(M) if values[j] > -math.inf),
                       key=lambda j: (not math.isnan(float(row[j])), -values[j], j))[:k]
        if (valid is not None and not bool(valid[i])) or not order:
            continue
        rows += 1
        units[i, :len(order)] = torch.tensor(order)
        e = torch.exp(row[order] - row[order[0]])
        shares[i, :len(order)] = e / e.sum()
        counts[order] += 1
        e = torch.exp(row - row[order[0]])
        probs += e / e.sum()
    probs = probs / max(1, rows)
    load = counts.to(F64) / max(1, int(counts.sum()))
    return units, shares, M * (load * probs).sum(), counts, probs, rows


def choose_units_backward(logits, k, d_shares, d_balance, valid=None):
    """``d_logits [n, M]`` by the formulas."""
    n, M = logits.shape
    units, shares, _, counts, _, rows = choose_units(logits, k, valid)
    load = counts.to(F64) / max(1, int(counts.sum()))
    d = torch.zeros(n, M, dtype=F64)
    for i in range(n):
        have = int((units[i] >= 0).sum())
        if not have:
            continue
        at, s = units[i, :have], shares[i, :have]
        if d_shares is not None:
            g = d_shares[i, :have].to(F64)
            d[i, at] += s * (g - (s * g).sum())
        if d_balance is not None:
            p = torch.softmax(logits[i].to(F64), dim=0)
            d[i] += float(d_balance) * M / rows * p * (load - (p * load).sum())
    return d


def grad_norm(grads):
    """The norm of all elements, by a compensated sum."""
    return math.sqrt(math.fsum(float(v) ** 2 for g in grads for v in g.reshape(-1).tolist()))


def clip_coefficient(norm, max_norm):
    if not math.isfinite(norm):
        return 1.0
    return min(1.0, max_norm / (norm + 1e-6))
