"""A small token model of routed layers: trained by distillation, then sampled from.

Each block mixes the sequence with the gated recurrence, whose gate and value are the two halves of
one TropLinear's output, and the head is a TropLinear over the vocabulary. The student learns a
teacher's top logits (here a fixed bigram table's) with the distillation loss, and generates with
one recurrence step and one sampling call a token.

    python examples/routed_sequence_model.py [--steps N]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn
from torch import Tensor

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tropnn_b200 import (  # noqa: E402
    TropLinear,
    distill_loss_b200,
    gated_recurrence_b200,
    gated_recurrence_step_b200,
    sample_tokens_b200,
)


class RoutedBlock(nn.Module):
    """x + out(recurrence(gate, value)), gate and value from one routed projection."""

    def __init__(self, dim: int, *, seed: int) -> None:
        super().__init__()
        self.dim = dim
        self.norm = nn.LayerNorm(dim)
        self.mix = TropLinear(dim, 2 * dim, heads=16, cells=4, code_dim=dim, seed=seed, cache_route_debug=False)
        self.out = TropLinear(dim, dim, heads=16, cells=4, code_dim=dim, seed=seed + 1, cache_route_debug=False)

    def forward(self, x: Tensor, state: Tensor | None, reset: Tensor | None) -> tuple[Tensor, Tensor]:
        mixed = self.mix(self.norm(x))
        h, last = gated_recurrence_b200(mixed[..., : self.dim], mixed[..., self.dim :], state, reset=reset)
        return x + self.out(h), last

    def step(self, x: Tensor, state: Tensor) -> Tensor:
        """One token a row ([batch, dim]); the state is updated in place."""
        mixed = self.mix(self.norm(x))[:, 0]
        h = gated_recurrence_step_b200(mixed[:, : self.dim], mixed[:, self.dim :], state)
        return x + self.out(h)[:, 0]


class RoutedSequenceModel(nn.Module):
    def __init__(self, vocab: int, dim: int = 128, depth: int = 2, *, seed: int = 0) -> None:
        super().__init__()
        torch.manual_seed(seed)
        self.embed = nn.Embedding(vocab, dim)
        self.blocks = nn.ModuleList(RoutedBlock(dim, seed=seed + 10 * i) for i in range(depth))
        self.norm = nn.LayerNorm(dim)
        self.head = TropLinear(dim, vocab, heads=16, cells=4, code_dim=dim, seed=seed + 7, cache_route_debug=False)

    def forward(
        self, tokens: Tensor, states: list[Tensor] | None = None, reset: Tensor | None = None
    ) -> tuple[Tensor, list[Tensor]]:
        """Logits ``[batch, steps, vocab]`` of whole sequences and each block's last state; ``reset``
        marks the tokens that start a document."""
        x, last = self.embed(tokens), []
        for i, block in enumerate(self.blocks):
            x, state = block(x, None if states is None else states[i], reset)
            last.append(state)
        return self.head(self.norm(x)), last

    @torch.no_grad()
    def generate(self, prompt: Tensor, uniforms: Tensor, **sampling: float) -> Tensor:
        """``uniforms.shape[1]`` tokens after ``prompt``: a prefill, then a step and a draw a token. A row
        whose logits are no distribution draws -1."""
        logits, states = self(prompt)
        logits, tokens = logits[:, -1], []
        for t in range(uniforms.shape[1]):
            tokens.append(sample_tokens_b200(logits, uniforms[:, t], **sampling))
            x = self.embed(tokens[-1].clamp(min=0))
            for block, state in zip(self.blocks, states):
                x = block.step(x, state)
            logits = self.head(self.norm(x))[:, 0]
        return torch.stack(tokens, dim=1)


class BigramTeacher:
    """Top logits of the next token after each token, from a fixed table."""

    def __init__(self, vocab: int, top: int, *, seed: int = 1) -> None:
        gen = torch.Generator().manual_seed(seed)
        table = 2.5 * torch.randn(vocab, vocab, generator=gen)
        self.logits, self.indices = (t.cuda() for t in table.topk(top, dim=1))

    def __call__(self, tokens: Tensor) -> tuple[Tensor, Tensor]:
        return self.logits[tokens], self.indices[tokens]

    def sequences(self, batch: int, steps: int, gen: torch.Generator) -> Tensor:
        tokens = torch.randint(self.logits.shape[0], (batch,), generator=gen, device="cuda")
        out = [tokens]
        for _ in range(steps - 1):
            pick = torch.multinomial(torch.softmax(self.logits[tokens], dim=1), 1, generator=gen)
            tokens = self.indices[tokens].gather(1, pick)[:, 0]
            out.append(tokens)
        return torch.stack(out, dim=1)


def train(model: RoutedSequenceModel, teacher: BigramTeacher, steps: int, *, batch: int = 16, length: int = 96) -> list[float]:
    """Distils the teacher into the model; returns the losses."""
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    gen = torch.Generator(device="cuda").manual_seed(0)
    losses = []
    for _ in range(steps):
        tokens = teacher.sequences(batch, length + 1, gen)
        reset = torch.rand(batch, length, generator=gen, device="cuda") < 1.0 / 32  # packed documents
        logits, _ = model(tokens[:, :-1], reset=reset)
        top_logits, top_indices = teacher(tokens[:, :-1])
        loss = distill_loss_b200(logits, top_logits, top_indices, tokens[:, 1:], temperature=2.0, label_weight=0.25)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    args = parser.parse_args()
    vocab = 200
    teacher = BigramTeacher(vocab, top=16)
    model = RoutedSequenceModel(vocab).cuda()
    losses = train(model, teacher, args.steps)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.3f}")
    print(f"last       loss {losses[-1]:.3f}")
    gen = torch.Generator(device="cuda").manual_seed(5)
    uniforms = torch.rand(2, 24, generator=gen, device="cuda")
    tokens = model.generate(teacher.sequences(2, 8, gen), uniforms, temperature=0.8, top_k=16, top_p=0.95)
    follows = (teacher.indices[tokens[:, :-1]] == tokens[:, 1:, None]).any(dim=2).float().mean()
    print(tokens.tolist())
    print(f"{100 * float(follows):.0f} percent of the drawn tokens are among the teacher's top {teacher.indices.shape[1]}")


if __name__ == "__main__":
    main()
