"""The language-model operators' definitions in float64 on the CPU, position by position and unit by
unit: the gated linear recurrence with its backward and its single position, the unit layer, and
the choice of a token. Test infrastructure only."""

from __future__ import annotations

import math

import torch

F64 = torch.float64


def gates(gate):
    """The share of the old state kept and the share written."""
    return 1 / (1 + torch.exp(gate)), 1 / (1 + torch.exp(-gate))


def scan_forward(y, gate, reset=None, h0=None, candidate="tanh"):
    """``(h [B, T, D], h_T [B, D])``."""
    y, gate = y.to(F64), gate.to(F64)
    B, T, D = y.shape
    c = torch.tanh(y) if candidate == "tanh" else y
    a, b = gates(gate)
    now = torch.zeros(B, D, dtype=F64) if h0 is None else h0.to(F64)
    h = torch.empty(B, T, D, dtype=F64)
    for t in range(T):
        if reset is not None:
            now = torch.where(reset[:, t, None], torch.zeros_like(now), now)
        now = a[:, t] * now + b[:, t] * c[:, t]
        h[:, t] = now
    return h, now


def scan_backward(y, gate, reset, h0, d_h, d_h_T, candidate="tanh"):
    """``(d_y, d_gate, d_h0)`` by the formulas, from the last position to the first."""
    y, gate = y.to(F64), gate.to(F64)
    B, T, D = y.shape
    c = torch.tanh(y) if candidate == "tanh" else y
    a, b = gates(gate)
    h, _ = scan_forward(y, gate, reset, h0, candidate)
    later = torch.zeros(B, D, dtype=F64) if d_h_T is None else d_h_T.to(F64)
    d_y, d_gate = torch.empty_like(y), torch.empty_like(y)
    for t in range(T - 1, -1, -1):
        old = h[:, t - 1] if t else (torch.zeros(B, D, dtype=F64) if h0 is None else h0.to(F64))
        drop = torch.zeros(B, 1, dtype=torch.bool) if reset is None else reset[:, t, None]
        old = torch.where(drop, torch.zeros_like(old), old)
        lam = later if d_h is None else later + d_h[:, t].to(F64)
        d_y[:, t] = lam * b[:, t] * ((1 - c[:, t] ** 2) if candidate == "tanh" else 1)
        d_gate[:, t] = lam * a[:, t] * b[:, t] * (c[:, t] - old)
        later = torch.where(drop, torch.zeros_like(lam), lam * a[:, t])
    return d_y, d_gate, later


def scan_step(y, gate, state, rows=None, reset=None, candidate="tanh"):
    """``(h [n, D], the pool afterwards)``; a row outside the pool is padding."""
    state = state.to(F64).clone()
    h = torch.zeros(y.shape, dtype=F64)
    for i in range(y.shape[0]):
        row = i if rows is None else int(rows[i])
        if not 0 <= row < state.shape[0]:
            continue
        one = None if reset is None else reset[i].reshape(1, 1)
        now = scan_forward(y[i].reshape(1, 1, -1), gate[i].reshape(1, 1, -1), one,
                           state[row].reshape(1, -1), candidate)[1][0]
        h[i] = state[row] = now
    return h, state


def unit_layer(x, router, W1, b1, W2, b2, k, activation="gelu"):
    """``y [n, d_out]``: the ``k`` largest router products of each token (ties: the lowest unit),
    their softmax, and the chosen units' outputs summed with it."""
    x, router, W1, W2 = (t.to(F64) for t in (x, router, W1, W2))
    n, H = x.shape[0], W2.shape[1]
    y = torch.zeros(n, W2.shape[2], dtype=F64)
    for i in range(n):
        logits = (router * x[i]).sum(1)
        chosen = sorted(range(len(logits)), key=lambda j: (-float(logits[j]), j))[:k]
        top = max(float(logits[j]) for j in chosen)
        share = [math.exp(float(logits[j]) - top) for j in chosen]
        for j, p in zip(chosen, share):
            z = x[i] @ W1[j]
            if b1 is not None:
                z = z + b1[j].to(F64)
            if activation == "gelu":
                z = 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
            else:
                z = z[:H] / (1 + torch.exp(-z[:H])) * z[H:]
            z = z @ W2[j]
            if b2 is not None:
                z = z + b2[j].to(F64)
            y[i] += p / sum(share) * z
    return y


def kept_tokens(logits, temperature, top_k, top_p, min_p):
    """One row's kept tokens with their weights ``exp((l - max) / t)``, in the order of their
    logits (ties: the lowest token): the first ``top_k``, of these the shortest prefix that holds
    ``top_p`` of their mass, of these those with at least ``min_p`` of the largest."""
    values = [float(v) for v in logits]
    values = [-math.inf if math.isnan(v) else v for v in values]
    best = max(values)
    if best == -math.inf:
        return []
    order = sorted((j for j, v in enumerate(values) if v > -math.inf),
                   key=lambda j: (-values[j], j))

    def weight(v):
        return 1.0 if v == best else math.exp(max((v - best) / temperature, -800.0))

    kept = [(j, weight(values[j])) for j in order][:top_k if top_k > 0 else None]
    if top_p < 1:
        total, before, prefix = sum(w for _, w in kept), 0.0, []
        for j, w in kept:
            if prefix and not before < top_p * total:
                break
            prefix.append((j, w))
            before += w
        kept = prefix
    return [kept[0]] + [(j, w) for j, w in kept[1:] if w >= min_p]


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(token, margin)`` of one row: the first kept token, in the order of tokens, at which the
    running mass exceeds ``u`` of the whole, and how far ``u`` is from the nearest place where the
    answer changes (a share of the mass). ``temperature <= 0``: the first largest logit."""
    values = [float(v) for v in logits]
    values = [-math.inf if math.isnan(v) else v for v in values]
    best = max(values)
    if best == -math.inf:
        return -1, 1.0
    if not temperature > 0:
        return values.index(best), 1.0
    kept = sorted(kept_tokens(logits, temperature, top_k, top_p, min_p))
    total, run, token, margin = sum(w for _, w in kept), 0.0, None, 1.0
    for j, w in kept:
        run += w
        margin = min(margin, abs(run / total - u)) if j != kept[-1][0] else margin
        if token is None and run > u * total:
            token = j
    return (kept[-1][0] if token is None else token), margin
