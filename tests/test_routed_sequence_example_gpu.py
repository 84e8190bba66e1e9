"""The example that runs the token operators together with the routed layers."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "routed_sequence_model.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("routed_sequence_model", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_student_learns_and_answers(example) -> None:
    teacher = example.BigramTeacher(60, top=8)
    model = example.RoutedSequenceModel(60, dim=64, depth=1).cuda()
    losses = example.train(model, teacher, 60, batch=8, length=48)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert sum(losses[-10:]) < 0.7 * sum(losses[:10])
    gen = torch.Generator(device="cuda").manual_seed(2)
    prompt, uniforms = teacher.sequences(3, 5, gen), torch.rand(3, 12, generator=gen, device="cuda")
    tokens = model.generate(prompt, uniforms, top_k=8, top_p=0.9)
    assert tokens.shape == (3, 12) and bool(((tokens >= 0) & (tokens < 60)).all())
    assert torch.equal(tokens, model.generate(prompt, uniforms, top_k=8, top_p=0.9))


def test_steps_follow_the_whole_sequence(example) -> None:
    """Logits of a token after a prefill and steps are those of the whole sequence: f32 layers whose sums
    run in another order for another number of rows (1e-5 of the values a layer, three layers on top of
    one another, and a route may flip only between scores that close)."""
    model = example.RoutedSequenceModel(60, dim=64, depth=1).cuda().eval()
    tokens = torch.randint(60, (4, 20), generator=torch.Generator().manual_seed(3)).cuda()
    with torch.no_grad():
        whole, _ = model(tokens)
        _, states = model(tokens[:, :12])
        for t in range(12, 20):
            x = model.embed(tokens[:, t])
            for block, state in zip(model.blocks, states):
                x = block.step(x, state)
            logits = model.head(model.norm(x))[:, 0]
            assert float((logits - whole[:, t]).abs().max()) <= 1e-3 * float(whole[:, t].abs().max())


def test_a_row_without_a_distribution_goes_on(example, monkeypatch) -> None:
    """The sampler's -1 is no row of the embedding."""
    model = example.RoutedSequenceModel(60, dim=64, depth=1).cuda().eval()
    monkeypatch.setattr(example, "sample_tokens_b200", lambda logits, u, **_: torch.full_like(u, -1, dtype=torch.int64))
    tokens = model.generate(torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.rand(2, 4, device="cuda"))
    assert bool((tokens == -1).all())
