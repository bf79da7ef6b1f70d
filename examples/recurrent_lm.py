"""A small recurrent language model on this package's operators, from training to answering.

The model reads tokens (:mod:`hsn_amd.embedding`) through the gated linear recurrence
(:mod:`hsn_amd.scan`) and answers through a bank of units that a router chooses (two a token):

    x = embed[token];  y | gate = x Wz;  h = scan(y, gate);  o = units(h);  logits = o out^T

Training runs whole windows: the recurrence as one autograd node with its state carried from window
to window, the units' choice with its balance loss (:mod:`hsn_amd.unit_router`), the units as the grouped
unit MLP of :mod:`hsn_amd.kernels.ops`, the loss from the tokens' log probabilities
(:mod:`hsn_amd.scoring`), and the gradients clipped by their global norm (:mod:`hsn_amd.grad_clip`).
Answering reads the prompt with one forward scan, and then takes a token at a time: one position of the
recurrence on a pool of states (:func:`hsn_amd.scan.step`), the unit layer for a few tokens
(:func:`hsn_amd.unit_layer.unit_layer`) and the choice of a token from given random numbers
(:func:`hsn_amd.sampling.sample`). The decoded position is a HIP graph, replayed for every token.

    python examples/recurrent_lm.py

trains it on a text of repeated phrases and prints how fast it answers.
"""

from __future__ import annotations

import sys
import time
from pathlib import Path

import torch
from torch import Tensor

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from hsn_amd import embedding, grad_clip, sampling, scan, scoring, unit_router
from hsn_amd.kernels import ops
from hsn_amd.unit_layer import unit_layer


class RecurrentLM(torch.nn.Module):
    """``d``-wide units (hidden ``H``, ``M`` of them, ``k`` a token) over ``4 d`` recurrent channels."""

    def __init__(self, vocabulary: int, d: int = 64, H: int = 512, M: int = 8, k: int = 2):
        super().__init__()
        D = 4 * d
        self.k, self.D = k, D

        def weight(*shape, scale):
            return torch.nn.Parameter(torch.randn(*shape) * scale)

        self.embed = weight(vocabulary, D, scale=0.3)
        self.Wz = weight(D, 2 * D, scale=D ** -0.5)
        self.router = weight(M, D, scale=D ** -0.5)
        self.W1, self.b1 = weight(M, D, H, scale=D ** -0.5), weight(M, H, scale=0.0)
        self.W2, self.b2 = weight(M, H, d, scale=H ** -0.5), weight(M, d, scale=0.0)
        self.out = weight(vocabulary, d, scale=d ** -0.5)

    def gates(self, tokens: Tensor) -> tuple[Tensor, Tensor]:
        z = embedding.embed(tokens, self.embed) @ self.Wz
        return z[..., :self.D], z[..., self.D:] - 1.0

    def forward(self, tokens: Tensor, reset: Tensor, h0: Tensor) -> tuple[Tensor, Tensor]:
        """``(logits [B, T, vocabulary], the state after the window)``, with a gradient."""
        logits, _, h_T = self.window(tokens, reset, h0)
        return logits, h_T

    def window(self, tokens: Tensor, reset: Tensor, h0: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        """The same with the units' balance loss (1 where all are chosen alike) between."""
        h, h_T = scan.gated_scan(*self.gates(tokens), reset, h0)
        flat = h.reshape(-1, self.D)
        units, share, balance, _ = unit_router.choose_units(flat @ self.router.t(), self.k)
        pairs = flat.repeat_interleave(self.k, dim=0)
        o, _ = ops.mlp_op(pairs, units.reshape(-1), self.W1, self.b1, self.W2, self.b2)
        o = (o.view(-1, self.k, o.shape[1]) * share[..., None]).sum(1)
        return (o @ self.out.t()).view(*tokens.shape, -1), balance, h_T

    def units(self, h: Tensor) -> Tensor:
        """The logits of a few tokens' states, without a gradient."""
        o = unit_layer(h, self.router, self.W1, self.b1, self.W2, self.b2, self.k)
        return o @ self.out.t()


class Answerer:
    """Answers ``n`` prompts at a time with the model's weights as they are: a pool of states, and one
    position as a graph."""

    def __init__(self, model: RecurrentLM, n: int, **settings):
        self.model, self.n, self.settings = model, n, settings
        device = model.embed.device
        self.state = torch.zeros(n, model.D, device=device)
        self.token = torch.zeros(n, dtype=torch.int64, device=device)
        self.u = torch.zeros(n, device=device)
        self.logits = None
        self._graph = None

    def _position(self) -> None:
        y, gate = self.model.gates(self.token)
        self.logits = self.model.units(scan.step(y, gate, self.state))
        self.token.copy_(sampling.sample(self.logits, self.u, **self.settings))

    @torch.no_grad()
    def answer(self, prompt: Tensor, u: Tensor) -> Tensor:
        """``[n, steps]`` tokens after ``prompt [n, T]``, ``u [steps, n]`` the random numbers."""
        y, gate = self.model.gates(prompt[:, :-1])
        read = scan.forward(y, gate, save=False)
        if self._graph is None:  # once eagerly, so that everything is loaded, then captured
            self._position()
            torch.cuda.synchronize()
            self._graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph):
                self._position()
        self.state.copy_(read["h_T"])
        self.token.copy_(prompt[:, -1])
        answer = torch.empty(self.n, u.shape[0], dtype=torch.int64, device=prompt.device)
        for t in range(u.shape[0]):
            self.u.copy_(u[t])
            self._graph.replay()
            answer[:, t] = self.token
        return answer


def phrases(rows: int, length: int, vocabulary: int, seed: int) -> tuple[Tensor, Tensor]:
    """Rows of phrases of five tokens, in any order, every one always ending alike; token 0 starts a
    document. Returns the tokens and where documents start."""
    g = torch.Generator().manual_seed(seed)
    book = torch.randint(1, vocabulary, (6, 5), generator=torch.Generator().manual_seed(7))
    picks = torch.randint(0, 6, (rows, length // 5 + 1), generator=g)
    tokens = book[picks].reshape(rows, -1)[:, :length]
    start = torch.rand(rows, length, generator=g) < 1 / 64
    return torch.where(start, 0, tokens), start


def train(model: RecurrentLM, steps: int, rows: int = 16, length: int = 256, windows: int = 2,
          seed: int = 0, balance_weight: float = 0.01, max_norm: float = 1.0) -> list[float]:
    """Trains on fresh text, ``windows`` carried windows a step; returns the losses (without the
    balance's)."""
    device = model.embed.device
    optimiser = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for step in range(steps):
        tokens, start = (t.to(device) for t in phrases(rows, windows * length + 1, 32, seed + step))
        state = torch.zeros(rows, model.D, device=device)
        total = balance = 0.0
        for w in range(windows):
            at = slice(w * length, (w + 1) * length)
            logits, load, state = model.window(tokens[:, at], start[:, at].contiguous(), state)
            target = tokens[:, at.start + 1:at.stop + 1]
            total = total - scoring.token_logprobs(logits, target)[0].mean()
            balance = balance + load
        optimiser.zero_grad()
        (total + balance_weight * balance).backward()
        grad_clip.clip([p.grad for p in model.parameters()], max_norm)
        optimiser.step()
        losses.append(float(total.detach()) / windows)
    return losses


def main() -> None:
    torch.manual_seed(0)
    model = RecurrentLM(32).cuda()
    losses = train(model, 60)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} nats a token")
    n, steps = 16, 200
    prompt = phrases(n, 64, 32, 1000)[0].cuda()
    answerer = Answerer(model, n, temperature=0.8, top_k=20, top_p=0.95)
    u = torch.rand(steps, n, device="cuda")
    answerer.answer(prompt, u)
    torch.cuda.synchronize()
    began = time.perf_counter()
    answer = answerer.answer(prompt, u)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - began
    print(f"{n} answers of {steps} tokens: {1e6 * seconds / steps:.1f} us a position, "
          f"{n * steps / seconds:.0f} tokens/s; the first: {answer[0, :20].tolist()}")


if __name__ == "__main__":
    main()
